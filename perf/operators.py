"""Performance cases: a paged MLA cache from step to step, and dense attention over it.

Around its sparse attention a serving program keeps a paged cache.  Each step
it does four things with it, and every case is one of them:

* ``table``  -- ``extend_block_table``: blocks for the step's new tokens, their
  slots and positions, from the requests' lengths;
* ``rotary`` -- ``rotary``: rotary positions on queries and indexer heads, both
  pair layouts, and the gradient;
* ``write``  -- ``write_kv_rows``: the new tokens' rows, rotated, into the cache,
  bf16 or fp8;
* ``shared`` -- ``forward_shared``: dense attention of a batch whose sequences
  share their first rows, over bf16 or fp8 caches, contiguous or paged.

``listed`` holds the measured cases, ``draw`` gives more of the same ranges,
``prepare``/``run`` make the inputs of a case and run one pass: the operator's
plain form in elementary torch operations, or with ``own`` the package's call.
``work`` counts what the pass cannot do without, ``exact`` computes its result
in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
LATENT, ROPE, FP8_ROW = 512, 64, 656
WIDTH = LATENT + ROPE
DEFAULT_SCALE = 1.0 / 24.0
MODEL_SCALE = 192.0 ** -0.5
MAX_SCORES = 4 * 512 * 128 * (8192 + 512)  # query rows x keys of the largest listed attention

ROTARY = dict(op="rotary", dtype="bf16", interleaved=True, start=0, transposed=False, yarn=False)
WRITE = dict(op="write", cache="bf16", interleaved=True, block=64)
SHARED = dict(op="shared", cache="bf16", block=0, causal=False, ragged=False, padded=False, model_scale=False)


def listed():
    """The measured cases."""
    return [
        # A decode step of 64 sequences, one new token each: some of them start a block.
        dict(op="table", name="table_decode_b64", batch=64, new=1, held=32767, ragged=True, block=64),
        # A step that admits 48 prompts of unequal length, small blocks.
        dict(op="table", name="table_prompts_b48", batch=48, new=2047, held=0, ragged=True, block=16),
        # The rotary part of 8 decode tokens' queries, a slice of the projected
        # 192-wide heads: launch latency.
        dict(ROTARY, name="rotary_decode_b8", tokens=8, heads=128, width=192, start=128, dim=64, far=32768, split=True),
        # The same for a 4096-token prompt chunk far into a long context.
        dict(ROTARY, name="rotary_prompt_h128", tokens=4096, heads=128, width=192, start=128, dim=64, far=131072,
             split=True, yarn=True),
        # The gradient of an indexer's rotated heads in training: half layout,
        # the first 64 of 128 dims, an odd number of tokens, 32 bits.
        dict(ROTARY, name="rotary_index_grad", tokens=1999, heads=64, width=128, dim=64, far=16384, split=False,
             dtype="f32", interleaved=False, transposed=True),
        # A decode step's new rows into a bf16 cache.
        dict(WRITE, name="write_decode_b33", tokens=33, far=32768, spare=16384),
        # A prompt's rows into an fp8 cache.
        dict(WRITE, name="write_prompt_fp8", tokens=8191, far=16384, spare=4096, cache="fp8"),
        # Three short requests behind a short system prompt, a slice of 16 heads,
        # contiguous cache, nothing aligned: latency.
        dict(SHARED, name="shared_small_h16", batch=3, queries=1, heads=16, prefix=500, suffix=301, ragged=True),
        # A tensor-parallel decode step of 64 requests on an fp8 paged cache
        # behind a long document.
        dict(SHARED, name="shared_decode_fp8_h16", batch=64, queries=1, heads=16, prefix=16384, suffix=2048, ragged=True,
             cache="fp8", block=64, model_scale=True),
        # Draft-and-verify of 16 requests with all heads, small blocks.
        dict(SHARED, name="shared_verify_h128", batch=16, queries=3, heads=128, prefix=8192, suffix=4096, ragged=True,
             block=16, causal=True, model_scale=True),
        # Prefill of six requests' own odd-length parts behind a shared prompt,
        # a slice of 32 heads; one request of the batch is padding.
        dict(SHARED, name="shared_suffix_h32", batch=6, queries=333, heads=32, prefix=4099, suffix=333, block=64,
             causal=True, padded=True),
        # The largest: the prompts of four requests behind one document, all heads.
        dict(SHARED, name="shared_suffix_h128", batch=4, queries=512, heads=128, prefix=8192, suffix=512, causal=True),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case of the listed ones' ranges: batches of 1 to 64, steps of 1
    to 65536 tokens, prefixes of up to 16384 rows and own parts of up to 4096."""
    op = rng.choices(["table", "rotary", "write", "shared"], [3, 4, 3, 8])[0]
    if op == "table":
        new = rng.choice([1, 1, rng.randint(2, 4), _log_int(rng, 8, 2048)])
        return dict(op=op, batch=_log_int(rng, 1, 64 if new > 64 else 256), new=new,
                    held=rng.choice([0, _log_int(rng, 1, 65536)]), ragged=rng.random() < 0.8,
                    block=rng.choice([16, 32, 64, 48]))
    if op == "rotary":
        heads = rng.choice([1, 16, 32, 64, 128])
        width = rng.choice([64, 128, 192])
        split = rng.random() < 0.5
        dim = 64 if split else rng.choice([64, min(width, 128), 32])
        return dict(ROTARY, tokens=_log_int(rng, 1, max(4096, min(65536, 4096 * 128 // heads // 4))), heads=heads,
                    width=width, start=rng.choice([0, width - dim]), dim=dim, far=_log_int(rng, 64, 1 << 20),
                    split=split, yarn=rng.random() < 0.5, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]),
                    interleaved=rng.random() < 0.5, transposed=rng.random() < 0.3)
    if op == "write":
        return dict(WRITE, tokens=_log_int(rng, 1, 32768), far=_log_int(rng, 64, 1 << 20), spare=_log_int(rng, 64, 16384),
                    cache=rng.choice(["bf16", "fp8"]), interleaved=rng.random() < 0.7, block=rng.choice([16, 64, 48]))
    decode = rng.random() < 0.6
    case = dict(SHARED, batch=_log_int(rng, 1, 64) if decode else rng.randint(1, 8),
                queries=rng.choice([1, 1, 2, 3, 4]) if decode else _log_int(rng, 8, 512),
                heads=rng.choice([16, 16, 32, 48, 64, 128]), prefix=rng.choice([0, _log_int(rng, 16, 16384)]),
                ragged=decode and rng.random() < 0.7, block=rng.choice([0, 16, 64, 48]),
                cache=rng.choice(["bf16", "bf16", "fp8"]), causal=True, model_scale=rng.random() < 0.5)
    case["suffix"] = case["queries"] + (_log_int(rng, 1, 4096) if decode else rng.choice([0, _log_int(rng, 1, 1024)]))
    while case["batch"] * case["queries"] * case["heads"] * (case["prefix"] + case["suffix"]) > MAX_SCORES:
        case["queries"] = (case["queries"] + 1) // 2
        case["batch"] = (case["batch"] + 1) // 2
    return dict(case, padded=case["batch"] > 1 and rng.random() < 0.3)


# ------------------------------------------------------------------ inputs

def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _normal(gen, *dims):
    return torch.randn(dims, generator=gen, device=DEVICE, dtype=torch.float32)


def _integers(gen, low, high, *dims):
    return torch.randint(low, high, dims, generator=gen, device=DEVICE)


def _shuffled(gen, n):
    return torch.randperm(n, generator=gen, device=DEVICE)


def _frequencies(dim, yarn):
    """Radians a position for each pair, 64 bits: theta 10000, or stretched 40
    times by the rule that leaves the fast pairs as they are."""
    i = torch.arange(dim // 2, dtype=torch.float64)
    freq = 10000.0 ** (-2.0 * i / dim)
    if yarn:
        border = [dim * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(10000.0)) for turns in (32.0, 1.0)]
        low, high = max(math.floor(border[0]), 0), min(math.ceil(border[1]), dim - 1)
        keep = 1.0 - ((i - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
        freq = freq / 40.0 * (1.0 - keep) + freq * keep
    return freq.to(DEVICE)


def _fp8_rows(kv, k_rope):
    """bf16 rows as 656 bytes: 512 e4m3 codes, four fp32 power-of-two scales, 64 bf16 rope values."""
    x = kv.float().unflatten(-1, (4, 128))
    scale = x.abs().amax(-1, keepdim=True) / 448.0
    mantissa, exponent = torch.frexp(torch.where(scale > 0, scale, torch.ones_like(scale)))
    scale = torch.ldexp(torch.ones_like(scale), exponent - (mantissa == 0.5).int())
    codes = (x / scale).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).flatten(-2)
    return torch.cat([codes.view(torch.uint8), scale.flatten(-2).view(torch.uint8),
                      k_rope.contiguous().view(torch.uint8)], -1)


def _prepare_table(case, gen):
    batch, new, held, block = case["batch"], case["new"], case["held"], case["block"]
    lengths, add = torch.full((batch,), held, device=DEVICE), torch.full((batch,), new, device=DEVICE)
    if case["ragged"]:
        lengths = _integers(gen, held // 2, held + 1, batch)
        if new > 4:
            add = _integers(gen, 0, new + 1, batch)
    wide = -(-(held + new) // block) + 3
    blocks = batch * wide
    order = _shuffled(gen, blocks).int()
    table = order.reshape(batch, wide).clone()
    in_use = torch.arange(wide, device=DEVICE) < (lengths + block - 1)[:, None] // block
    free = table.masked_select(~in_use)[_shuffled(gen, int((~in_use).sum()))].contiguous()
    return dict(table=table.masked_fill(~in_use, -1).contiguous(), lengths=lengths.int(), add=add.int(), free=free,
                block=block, max_tokens=batch * new)


DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _prepare_rotary(case, gen):
    """``split``: the rotated part goes, alone, to a new tensor (queries are
    projected with both parts in one row); else whole heads are rewritten."""
    tokens, dim, start = case["tokens"], case["dim"], case["start"]
    first = int(_integers(gen, 0, max(1, case["far"] - tokens), 1))
    x = _normal(gen, tokens, case["heads"], case["width"]).to(DTYPES[case["dtype"]])
    return dict(x=x[..., start:start + dim] if case["split"] else x, start=0 if case["split"] else start, dim=dim,
                positions=(torch.arange(tokens, device=DEVICE) + first).int(), frequencies=_frequencies(dim, case["yarn"]),
                interleaved=case["interleaved"], transposed=case["transposed"])


def _prepare_write(case, gen):
    """The latent and the rotary part as a model has them: one normalised, one
    still in the row that the projection made."""
    tokens, block = case["tokens"], case["block"]
    blocks = -(-(tokens + case["spare"]) // block)
    row = _normal(gen, tokens, WIDTH).bfloat16()
    gain = torch.exp(_normal(gen, LATENT))
    state = dict(kv=(_normal(gen, tokens, LATENT) * gain).bfloat16(), k_rope=row[:, LATENT:],
                 slots=_shuffled(gen, blocks * block)[:tokens].int(), fp8=case["cache"] == "fp8",
                 positions=(torch.arange(tokens, device=DEVICE) + int(_integers(gen, 0, case["far"], 1))).int(),
                 frequencies=_frequencies(ROPE, False), interleaved=case["interleaved"])
    if state["fp8"]:
        state["cache"] = torch.zeros((blocks, block, 1, FP8_ROW), device=DEVICE, dtype=torch.uint8)
    else:
        state["cache"] = torch.zeros((blocks, block, 1, LATENT), device=DEVICE, dtype=torch.bfloat16)
        state["rope_cache"] = torch.zeros((blocks, block, 1, ROPE), device=DEVICE, dtype=torch.bfloat16)
    return state


def _prepare_shared(case, gen):
    batch, queries, heads, block = case["batch"], case["queries"], case["heads"], case["block"]
    prefix, context = case["prefix"], case["prefix"] + case["suffix"]
    state = dict(q=_normal(gen, batch, queries, heads, LATENT).bfloat16(), prefix=prefix, block_table=None,
                 q_rope=_normal(gen, batch, queries, heads, ROPE).bfloat16(),
                 scale=MODEL_SCALE if case["model_scale"] else None)
    if block:
        # the prefix's whole blocks are the same in every row of the table
        whole, wide = prefix // block, -(-context // block)
        context = wide * block
        blocks = whole + batch * (wide - whole)
        order = _shuffled(gen, blocks).int()
        state["block_table"] = torch.cat([order[:whole].expand(batch, -1),
                                          order[whole:].reshape(batch, wide - whole)], 1).contiguous()
        lead = (blocks, block, 1)
    else:
        lead = (batch, context, 1)
    kv, k_rope = _normal(gen, *lead, LATENT).bfloat16(), _normal(gen, *lead, ROPE).bfloat16()
    # rows of the prefix that lie outside its whole blocks are held by every sequence
    if block and prefix % block:
        tail = state["block_table"][:, whole].long()
        kv[tail, :prefix % block] = kv[tail[:1], :prefix % block].clone()
        k_rope[tail, :prefix % block] = k_rope[tail[:1], :prefix % block].clone()
    if not block:
        kv[:, :prefix] = kv[:1, :prefix].clone()
        k_rope[:, :prefix] = k_rope[:1, :prefix].clone()
    state["kv"], state["k_rope"] = (_fp8_rows(kv, k_rope), None) if case["cache"] == "fp8" else (kv, k_rope)
    seen = torch.full((batch, 1), prefix + case["suffix"], device=DEVICE)
    if case["ragged"]:
        seen = seen - _integers(gen, 0, max(1, case["suffix"] - queries + 1), batch, 1)
    seen = seen - (queries - 1 - torch.arange(queries, device=DEVICE) if case["causal"] else 0)
    seen = seen.expand(batch, queries).clone()
    if case["padded"]:
        seen[batch - 1] = 0
    state["lengths"] = seen.int()
    return state


def prepare(case, seed):
    gen = _generator(seed)
    make = {"table": _prepare_table, "rotary": _prepare_rotary, "write": _prepare_write, "shared": _prepare_shared}
    return dict(make[case["op"]](case, gen), op=case["op"])


# ------------------------------------------------------------------ plain forms

def _plain_table(s):
    table, block, free = s["table"], s["block"], s["free"].long()
    held, add = s["lengths"].long(), s["add"].long()
    total = held + add
    first_new = (held + block - 1) // block
    need = (total + block - 1) // block - first_new
    zero = torch.zeros(1, device=table.device, dtype=torch.int64)
    starts, taken = torch.cat([zero, add.cumsum(0)]), torch.cat([zero, need.cumsum(0)])
    column = torch.arange(table.shape[1], device=table.device) - first_new[:, None]
    source = (taken[:-1, None] + column).clamp(0, free.numel() - 1)
    table.copy_(torch.where((column >= 0) & (column < need[:, None]), free[source].int(), table))
    token = torch.arange(s["max_tokens"], device=table.device)
    sequence = (token[:, None] >= starts[None, 1:]).sum(1)
    there = sequence < held.numel()
    sequence = sequence.clamp_max(held.numel() - 1)
    position = held[sequence] + token - starts[sequence]
    entry = table[sequence, (position // block).clamp(0, table.shape[1] - 1)].long()
    slots = torch.where(there, entry * block + position % block, -1).int()
    return table, slots, torch.where(there, position, 0).int(), starts.int(), total.int(), taken[-1:].int()


def _turn(x, positions, frequencies, interleaved, back):
    """x [tokens, ..., dim] rotated, 32 bits; the angles are formed in 64."""
    angle = positions.double()[:, None] * frequencies
    cos, sin = angle.cos().float(), angle.sin().float()
    sin = -sin if back else sin
    if x.dim() == 3:
        cos, sin = cos[:, None], sin[:, None]
    x = x.float()
    pair = x.unflatten(-1, (-1, 2)).unbind(-1) if interleaved else x.unflatten(-1, (2, -1)).unbind(-2)
    turned = [pair[0] * cos - pair[1] * sin, pair[0] * sin + pair[1] * cos]
    return torch.stack(turned, -1 if interleaved else -2).flatten(-2)


def _plain_rotary(s):
    x, start, end = s["x"], s["start"], s["start"] + s["dim"]
    turned = _turn(x[..., start:end], s["positions"], s["frequencies"], s["interleaved"], s["transposed"])
    return torch.cat([x[..., :start], turned.to(x.dtype), x[..., end:]], -1)


def _plain_write(s):
    slots = s["slots"].long()
    rope = _turn(s["k_rope"], s["positions"], s["frequencies"], s["interleaved"], False).bfloat16()
    if s["fp8"]:
        s["cache"].view(-1, FP8_ROW)[slots] = _fp8_rows(s["kv"], rope)
    else:
        s["cache"].view(-1, LATENT)[slots] = s["kv"]
        s["rope_cache"].view(-1, ROPE)[slots] = rope
    return _cache_values(s)


def _cache_values(s):
    """The caches as values: an fp8 row's codes, scales and rope values are views of its bytes."""
    if not s["fp8"]:
        return s["cache"], s["rope_cache"]
    rows = s["cache"].view(-1, FP8_ROW)
    return (rows[:, :LATENT].view(torch.float8_e4m3fn), rows[:, LATENT:LATENT + 16].view(torch.float32),
            rows[:, LATENT + 16:].view(torch.bfloat16))


def _rows(s, flat):
    """Cache rows [n, 576] of the flat row numbers, 32 bits."""
    kv = s["kv"].view(-1, s["kv"].shape[-1])[flat]
    if s["k_rope"] is not None:
        return torch.cat([kv, s["k_rope"].view(-1, ROPE)[flat]], -1).float()
    codes = kv[..., :LATENT].contiguous().view(torch.float8_e4m3fn).float()
    scale = kv[..., LATENT:LATENT + 16].contiguous().view(torch.float32)
    latent = (codes.unflatten(-1, (4, 128)) * scale[..., None]).flatten(-2)
    return torch.cat([latent, kv[..., LATENT + 16:].contiguous().view(torch.bfloat16).float()], -1)


def _plain_shared(s):
    batch, queries, heads, _ = s["q"].shape
    prefix, table = s["prefix"], s["block_table"]
    if table is None:
        context = s["kv"].shape[1]
        flat = torch.arange(batch * context, device=DEVICE).view(batch, context)
    else:
        block = s["kv"].shape[1]
        flat = (table.long()[:, :, None] * block + torch.arange(block, device=DEVICE)).flatten(1)
        context = flat.shape[1]
    shared, private = _rows(s, flat[0, :prefix]), _rows(s, flat[:, prefix:])
    q = torch.cat([s["q"], s["q_rope"]], -1).float().view(batch, queries * heads, WIDTH)
    score = torch.cat([(q.view(-1, WIDTH) @ shared.t()).view(batch, queries * heads, prefix),
                       torch.bmm(q, private.transpose(1, 2).contiguous())], -1)
    score = score.view(batch, queries, heads, context) * (DEFAULT_SCALE if s["scale"] is None else s["scale"])
    hidden = torch.arange(context, device=DEVICE) >= s["lengths"][..., None, None]
    score = score.masked_fill(hidden, -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = torch.exp(score - top.clamp_min(torch.finfo(torch.float32).min))
    total = weight.sum(-1, keepdim=True)
    weight = (weight / torch.where(total > 0, total, 1.0)).view(batch, queries * heads, context)
    latent = ((weight[..., :prefix].reshape(q.numel() // WIDTH, prefix) @ shared[:, :LATENT]).view(batch, queries * heads, LATENT)
              + torch.bmm(weight[..., prefix:], private[..., :LATENT].contiguous()))
    shape = (batch, 1, queries, heads)
    return latent.view(batch, queries, heads, LATENT).bfloat16(), top.view(shape), total.view(shape)


# ------------------------------------------------------------------ one pass

def run(state):
    op = state["op"]
    if not own:
        plain = {"table": _plain_table, "rotary": _plain_rotary, "write": _plain_write, "shared": _plain_shared}
        return plain[op](state)
    import dsa_amd

    s = state
    if op == "table":
        return (s["table"], *dsa_amd.extend_block_table(s["table"], s["lengths"], s["add"], s["free"], s["block"],
                                                        s["max_tokens"]))
    if op == "rotary":
        return dsa_amd.rotary(s["x"], s["positions"], s["frequencies"], interleaved=s["interleaved"], start=s["start"],
                              transposed=s["transposed"])
    if op == "write":
        dsa_amd.write_kv_rows(s["kv"], s["k_rope"], s["slots"], s["cache"], s.get("rope_cache"),
                              positions=s["positions"], frequencies=s["frequencies"], interleaved=s["interleaved"])
        return _cache_values(s)
    return dsa_amd.forward_shared(s["q"], s["kv"], s["q_rope"], s["k_rope"], s["lengths"], s["prefix"],
                                  scale=s["scale"], block_table=s["block_table"])


# ------------------------------------------------------------------ bounds

def work(case):
    """Bytes and operations of one pass: each input read once, each output written once."""
    op = case["op"]
    if op == "table":
        tokens = case["batch"] * case["new"] // (2 if case["ragged"] and case["new"] > 4 else 1)
        return {"bytes": 8 * case["batch"] * case["new"] + 8 * (tokens // case["block"]) + 16 * case["batch"],
                "flops": 0}
    if op == "rotary":
        size = 4 if case["dtype"] == "f32" else 2
        values = case["tokens"] * case["heads"] * (case["dim"] if case["split"] else case["width"])
        return {"bytes": 2 * size * values + 4 * case["tokens"],
                "flops": 3 * case["tokens"] * case["heads"] * case["dim"]}
    if op == "write":
        return {"bytes": case["tokens"] * (2 * WIDTH + (FP8_ROW if case["cache"] == "fp8" else 2 * WIDTH) + 8),
                "flops": 3 * case["tokens"] * ROPE}
    live = max(1, case["batch"] - (1 if case["padded"] else 0))
    suffix = case["suffix"] - ((case["suffix"] - case["queries"]) // 2 if case["ragged"] else 0)
    keys = case["prefix"] + suffix - ((case["queries"] - 1) / 2 if case["causal"] else 0)
    rows = live * case["queries"] * case["heads"]
    cached = case["prefix"] + live * suffix
    return {"bytes": (cached * (FP8_ROW if case["cache"] == "fp8" else 2 * WIDTH)
                      + case["batch"] * case["queries"] * case["heads"] * (2 * WIDTH + 2 * LATENT + 8)),
            "flops": 2 * rows * keys * (WIDTH + LATENT)}


# ------------------------------------------------------------------ 64 bits

def _exact_table(s):
    """Sequence by sequence, on the host."""
    table, block, free = s["table"].tolist(), s["block"], iter(s["free"].tolist())
    starts, totals, slots, positions, taken = [0], [], [], [], 0
    for row, held, add in zip(table, s["lengths"].tolist(), s["add"].tolist()):
        for at in range(held, held + add):
            column = at // block
            if at % block == 0:
                row[column] = next(free)
                taken += 1
            slots.append(row[column] * block + at % block)
            positions.append(at)
        starts.append(starts[-1] + add)
        totals.append(held + add)
    rest = s["max_tokens"] - len(slots)
    return tuple(torch.tensor(v, dtype=torch.int32) for v in (table, slots + [-1] * rest, positions + [0] * rest, starts,
                                                              totals, [taken]))


def _exact_turn(x, positions, frequencies, interleaved, back):
    """As a product of complex numbers."""
    angle = positions.double()[:, None] * frequencies * (-1.0 if back else 1.0)
    turn = torch.polar(torch.ones_like(angle), angle).view(-1, *([1] * (x.dim() - 2)), angle.shape[1])
    half = angle.shape[1]
    x = x.double()
    z = torch.complex(x[..., 0::2], x[..., 1::2]) if interleaved else torch.complex(x[..., :half], x[..., half:])
    z = z * turn
    out = torch.empty_like(x)
    if interleaved:
        out[..., 0::2], out[..., 1::2] = z.real, z.imag
    else:
        out[..., :half], out[..., half:] = z.real, z.imag
    return out


def _exact_shared(s):
    """Sequence by sequence over its whole context."""
    batch, queries, heads, _ = s["q"].shape
    scale = DEFAULT_SCALE if s["scale"] is None else s["scale"]
    out = torch.zeros((batch, queries, heads, LATENT), device=DEVICE, dtype=torch.float64)
    peak = torch.full((batch, 1, queries, heads), -math.inf, device=DEVICE, dtype=torch.float64)
    total = torch.zeros_like(peak)
    for b in range(batch):
        seen = s["lengths"][b].long()
        most = int(seen.max())
        if most == 0:
            continue
        key = torch.arange(most, device=DEVICE)
        if s["block_table"] is None:
            flat = b * s["kv"].shape[1] + key
        else:
            block = s["kv"].shape[1]
            flat = s["block_table"][b].long()[key // block] * block + key % block
        rows = _rows(s, flat).double()
        step = max(1, (1 << 28) // (heads * most))
        for i in range(0, queries, step):
            q = torch.cat([s["q"][b, i:i + step], s["q_rope"][b, i:i + step]], -1).double()
            score = (q.flatten(0, 1) @ rows.t()).view(q.shape[0], heads, most) * scale
            score.masked_fill_(key >= seen[i:i + step, None, None], -math.inf)
            top = score.amax(-1)
            weight = torch.exp(score - top[..., None])
            norm = weight.sum(-1)
            out[b, i:i + step] = (weight.flatten(0, 1) @ rows[:, :LATENT]).view(q.shape[0], heads, LATENT) / norm[..., None]
            peak[b, 0, i:i + step], total[b, 0, i:i + step] = top, norm
    return out, peak, total


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "table":
        return _exact_table(s)
    if case["op"] == "shared":
        return _exact_shared(s)
    if case["op"] == "rotary":
        start, end = s["start"], s["start"] + s["dim"]
        out = s["x"].double()
        out[..., start:end] = _exact_turn(s["x"][..., start:end], s["positions"], s["frequencies"], s["interleaved"],
                                          s["transposed"])
        return out
    rope = _exact_turn(s["k_rope"], s["positions"], s["frequencies"], s["interleaved"], False)
    slots = s["slots"].long()
    if not s["fp8"]:
        kv, rotated = s["cache"].double().view(-1, LATENT), s["rope_cache"].double().view(-1, ROPE)
        kv[slots], rotated[slots] = s["kv"].double(), rope
        return kv.view(s["cache"].shape), rotated.view(s["rope_cache"].shape)
    count = s["cache"].numel() // FP8_ROW
    codes = torch.zeros((count, LATENT), device=DEVICE, dtype=torch.float64)
    scales = torch.zeros((count, 4), device=DEVICE, dtype=torch.float64)
    rotated = torch.zeros((count, ROPE), device=DEVICE, dtype=torch.float64)
    x = s["kv"].double().unflatten(-1, (4, 128))
    scale = torch.exp2(torch.ceil(torch.log2(x.abs().amax(-1) / 448.0)))
    codes[slots], scales[slots], rotated[slots] = (x / scale[..., None]).flatten(-2), scale, rope
    return codes, scales, rotated
