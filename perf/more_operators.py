"""Performance cases: a layer's way into the cache's attention, and a step that verifies drafted tokens.

Around its attention a model's layer normalises the residual stream, projects
it with 8-bit weights, and normalises the latent and the query again; a step
that verifies drafted tokens attends with a tree of them behind each sequence's
cache.  Every case is one of these:

* ``norm``    -- ``rms_norm``: root-mean-square norm with the residual's addition,
  and in training its gradients;
* ``codes``   -- ``rms_norm_fp8`` and ``quantize_fp8``: the same, or no norm at all,
  with an output of 8-bit codes and a scale for each 128 of them;
* ``product`` -- ``matmul_fp8``: the product of 8-bit rows with 8-bit weights that
  have a scale for each block of 128 by 128;
* ``tree``    -- ``draft_tree`` and ``forward_tree``: ancestors and positions of
  drafted tokens, and their dense attention over the cache, bf16 or fp8,
  contiguous or paged.

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
BLOCK = 128  # values that share a scale
E4M3_MAX = 448.0
EPS = 1e-6
DEFAULT_SCALE = 1.0 / 24.0
MODEL_SCALE = 192.0 ** -0.5
MAX_SCORES = 16 * 60 * 128 * (8192 + 60)  # query rows x keys of the largest listed attention
MAX_PRODUCT = 8192 * 16384 * 7168         # multiplications of the largest listed product
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}

NORM = dict(op="norm", dtype="bf16", width=0, residual=False, grad=False)
CODES = dict(op="codes", norm=True, residual=False, pow2=True)
PRODUCT = dict(op="product", dtype="bf16")
TREE = dict(op="tree", cache="bf16", block=0, prefix=0, ragged=False, padded=False, model_scale=False)


def listed():
    """The measured cases."""
    return [
        # The residual stream of 8 decode tokens between two layers: latency.
        dict(NORM, name="norm_decode_b8", tokens=8, dim=7168, residual=True),
        # A prompt chunk's cache latents: the first 512 of the projection's 576-wide rows.
        dict(NORM, name="norm_latent_prompt", tokens=4096, dim=512, width=576),
        # Training: the norm in front of a layer and all its gradients, an odd number of tokens.
        dict(NORM, name="norm_train", tokens=4095, dim=4096, residual=True, grad=True),
        # A verify step's residual stream on its way into 8-bit projections.
        dict(CODES, name="codes_verify_b64", tokens=192, dim=7168, residual=True),
        # A prompt's attention output, 128 heads of 128 values, in front of the output projection.
        dict(CODES, name="codes_prompt_heads", tokens=4095, dim=16384, norm=False, pow2=False),
        # The projections to query and cache latents (1536 and 576 side by side) of 8 decode tokens.
        dict(PRODUCT, name="product_decode_m8", rows=8, cols=2112, inner=7168),
        # The heads' queries (128 of 192) of a verify step, an odd number of tokens.
        dict(PRODUCT, name="product_verify_m77", rows=77, cols=24576, inner=1536),
        # The same latents as in the first of these, of a prompt chunk that ends inside a tile.
        dict(PRODUCT, name="product_chunk_m1000", rows=1000, cols=2112, inner=7168),
        # The largest: a prompt's output projection.
        dict(PRODUCT, name="product_prompt_m8192", rows=8192, cols=7168, inner=16384),
        # Three short requests with seven drafted tokens each, a slice of 16 heads, nothing aligned: latency.
        dict(TREE, name="tree_small_h16", batch=3, drafts=7, heads=16, context=777, ragged=True),
        # A tensor-parallel verify step of 32 requests on an fp8 paged cache behind a shared prompt; one is padding.
        dict(TREE, name="tree_fp8_h16", batch=32, drafts=33, heads=16, prefix=2048, context=8192, ragged=True,
             cache="fp8", block=64, padded=True, model_scale=True),
        # Large trees of 16 requests, all heads, small blocks.
        dict(TREE, name="tree_h128", batch=16, drafts=60, heads=128, context=8192, block=16, ragged=True,
             model_scale=True),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case of the listed ones' ranges: 1 to 16384 tokens of 64 to 16384
    values, products of up to 8192 rows, batches of 1 to 64 sequences with 1 to
    100 drafted tokens behind up to 16384 rows."""
    op = rng.choices(["norm", "codes", "product", "tree"], [4, 3, 6, 6])[0]
    if op == "norm":
        dim = rng.choice([512, 1536, 4096, 7168, _log_int(rng, 64, 8192)])
        case = dict(NORM, dim=dim, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), residual=rng.random() < 0.6,
                    grad=rng.random() < 0.4)
        case["tokens"] = _log_int(rng, 1, 4095 * 4096 // (dim if case["dtype"] != "f32" else 2 * dim))
        if not case["residual"] and rng.random() < 0.5:
            case["width"] = dim + rng.choice([8, 64, rng.randint(1, 100)])
        return case
    if op == "codes":
        dim = rng.choice([512, 1536, 7168, 16384, 16 * _log_int(rng, 4, 1024)])
        norm = rng.random() < 0.6
        return dict(CODES, dim=dim, norm=norm, residual=norm and rng.random() < 0.6, pow2=rng.random() < 0.5,
                    tokens=_log_int(rng, 1, min(16384, 4095 * 16384 // dim // (2 if norm else 1))))
    if op == "product":
        case = dict(PRODUCT, rows=rng.choice([_log_int(rng, 1, 128), _log_int(rng, 1, 8192)]),
                    cols=rng.choice([512, 2112, 7168, 24576, _log_int(rng, 16, 16384)]),
                    inner=rng.choice([512, 1536, 7168, 16384, 16 * _log_int(rng, 4, 1024)]),
                    dtype=rng.choice(["bf16", "bf16", "f16", "f32"]))
        while case["rows"] * case["cols"] * case["inner"] > MAX_PRODUCT:
            case["rows"] = (case["rows"] + 1) // 2
        return case
    case = dict(TREE, batch=_log_int(rng, 1, 64), drafts=rng.choice([1, _log_int(rng, 2, 16), _log_int(rng, 8, 100)]),
                heads=rng.choice([16, 16, 32, 48, 64, 128]), context=_log_int(rng, 16, 16384), ragged=rng.random() < 0.7,
                cache=rng.choice(["bf16", "bf16", "fp8"]), block=rng.choice([0, 16, 64, 48]),
                model_scale=rng.random() < 0.5)
    while case["batch"] * case["drafts"] * case["heads"] * (case["context"] + case["drafts"]) > MAX_SCORES:
        case["batch"] = (case["batch"] + 1) // 2
    if rng.random() < 0.4:
        case["prefix"] = rng.randint(1, max(1, case["context"] // 2))
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


def _stream(gen, tokens, dim):
    """A residual stream: some channels are a few times larger than the rest."""
    return _normal(gen, tokens, dim) * torch.exp(0.5 * _normal(gen, dim))


def _prepare_norm(case, gen):
    tokens, dim, dtype = case["tokens"], case["dim"], DTYPES[case["dtype"]]
    state = dict(x=_stream(gen, tokens, case["width"] or dim).to(dtype)[:, :dim], residual=None, grad=case["grad"],
                 weight=(1.0 + 0.2 * _normal(gen, dim)).to(dtype))
    if case["residual"]:
        state["residual"] = _stream(gen, tokens, dim).to(dtype)
    if case["grad"]:
        for name in ("x", "residual", "weight"):
            if state[name] is not None:
                state[name].requires_grad_(True)
        state["given"] = tuple(_normal(gen, tokens, dim).to(dtype) for _ in range(2 if case["residual"] else 1))
    return state


def _prepare_codes(case, gen):
    tokens, dim = case["tokens"], case["dim"]
    return dict(x=_stream(gen, tokens, dim).bfloat16(), pow2=case["pow2"],
                weight=(1.0 + 0.2 * _normal(gen, dim)).bfloat16() if case["norm"] else None,
                residual=_stream(gen, tokens, dim).bfloat16() if case["residual"] else None)


def _prepare_product(case, gen):
    """Activations with a scale for each row's 128 values, weights with one for
    each 128 by 128, both as large as their codes' range allows."""
    rows, cols, inner = case["rows"], case["cols"], case["inner"]
    blocks, bands = -(-inner // BLOCK), -(-cols // BLOCK)
    x = torch.nn.functional.pad(_stream(gen, rows, inner), (0, blocks * BLOCK - inner)).view(rows, blocks, BLOCK)
    a_scales = x.abs().amax(-1) / E4M3_MAX
    a = (x / a_scales[..., None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(rows, -1)[:, :inner].contiguous()
    b = torch.empty((cols, inner), device=DEVICE, dtype=torch.float8_e4m3fn)
    b_scales = torch.empty((bands, blocks), device=DEVICE, dtype=torch.float32)
    step = 32 * BLOCK  # of many columns, some at a time
    for first in range(0, cols, step):
        n = min(step, cols - first)
        high = -(-n // BLOCK)
        w = torch.zeros((high * BLOCK, blocks * BLOCK), device=DEVICE)
        w[:n, :inner] = _normal(gen, n, inner) * inner ** -0.5
        w = w.view(high, BLOCK, blocks, BLOCK)
        scale = w.abs().amax((1, 3)) / E4M3_MAX
        w = (w / scale[:, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX).view(high * BLOCK, -1)
        b[first:first + n] = w[:n, :inner].to(torch.float8_e4m3fn)
        b_scales[first // BLOCK:first // BLOCK + high] = scale
    return dict(a=a, a_scales=a_scales.contiguous(), b=b, b_scales=b_scales, dtype=DTYPES[case["dtype"]])


def _fp8_rows(kv, k_rope):
    """bf16 rows as 656 bytes: 512 e4m3 codes, four fp32 power-of-two scales, 64 bf16 rope values."""
    x = kv.float().unflatten(-1, (4, 128))
    scale = torch.exp2(torch.ceil(torch.log2(x.abs().amax(-1, keepdim=True) / E4M3_MAX)))
    codes = (x / scale).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).flatten(-2)
    return torch.cat([codes.view(torch.uint8), scale.flatten(-2).view(torch.uint8),
                      k_rope.contiguous().view(torch.uint8)], -1)


def _prepare_tree(case, gen):
    """Token t of a tree follows an earlier one, mostly a late one, or the
    context itself; a sequence that drafted fewer has -2 behind them."""
    batch, drafts, heads, block = case["batch"], case["drafts"], case["heads"], case["block"]
    prefix, context = case["prefix"], case["context"]
    state = dict(q=_normal(gen, batch, drafts, heads, LATENT).bfloat16(), prefix=prefix, block_table=None,
                 q_rope=_normal(gen, batch, drafts, heads, ROPE).bfloat16(),
                 scale=MODEL_SCALE if case["model_scale"] else None)
    token = torch.arange(drafts, device=DEVICE)
    back = torch.rand((batch, drafts), generator=gen, device=DEVICE).pow(3) * (token + 1)
    state["parents"] = (token - 1 - back.long()).clamp_min(-1).int()
    lengths = torch.full((batch,), context, device=DEVICE)
    if case["ragged"]:
        lengths = lengths - _integers(gen, 0, (context - prefix) // 2 + 1, batch)
        held = _integers(gen, (drafts + 1) // 2, drafts + 1, batch, 1)
        state["parents"] = state["parents"].masked_fill(token >= held, -2)
    if case["padded"]:
        lengths[batch - 1] = 0
        state["parents"][batch - 1] = -2
    state["lengths"] = lengths.int()
    total = context + drafts
    if block:  # the prefix's whole blocks are the same in every row of the table
        whole, wide = prefix // block, -(-total // block)
        blocks = whole + batch * (wide - whole)
        order = _shuffled(gen, blocks).int()
        state["block_table"] = torch.cat([order[:whole].expand(batch, -1),
                                          order[whole:].reshape(batch, wide - whole)], 1).contiguous()
        lead = (blocks, block, 1)
    else:
        lead = (batch, total, 1)
    kv, k_rope = _normal(gen, *lead, LATENT).bfloat16(), _normal(gen, *lead, ROPE).bfloat16()
    state["kv"], state["k_rope"] = (_fp8_rows(kv, k_rope), None) if case["cache"] == "fp8" else (kv, k_rope)
    return state


def prepare(case, seed):
    gen = _generator(seed)
    make = {"norm": _prepare_norm, "codes": _prepare_codes, "product": _prepare_product, "tree": _prepare_tree}
    return dict(make[case["op"]](case, gen), op=case["op"])


# ------------------------------------------------------------------ plain forms

def _add(s):
    """The stream behind the addition, as it is kept: rounded to its type."""
    return s["x"] if s["residual"] is None else (s["x"].float() + s["residual"].float()).to(s["x"].dtype)


def _normed(h, weight):
    h = h.float()
    return h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) * weight.float()


def _plain_norm(s):
    with torch.no_grad():
        h = _add(s)
        outputs = [_normed(h, s["weight"]).to(h.dtype)] + ([] if s["residual"] is None else [h])
        if s["grad"]:
            x, weight, given = h.float(), s["weight"].float(), s["given"][0].float()
            inverse = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
            unit = x * inverse
            back = given * weight
            dx = (back - unit * (back * unit).mean(-1, keepdim=True)) * inverse
            if s["residual"] is not None:
                dx = dx + s["given"][1].float()
            dx = dx.to(h.dtype)
            outputs += [dx] + ([] if s["residual"] is None else [dx]) + [(given * unit).sum(0).to(h.dtype)]
    return tuple(outputs)


def _plain_codes(s):
    h = _add(s)
    v = h.float() if s["weight"] is None else _normed(h, s["weight"])
    tokens, dim = v.shape
    blocks = -(-dim // BLOCK)
    v = torch.cat([v, v.new_zeros((tokens, blocks * BLOCK - dim))], -1).view(tokens, blocks, BLOCK)
    top = v.abs().amax(-1, keepdim=True)
    scale = torch.where(top > 0, top / E4M3_MAX, 1.0)
    if s["pow2"]:
        mantissa, exponent = torch.frexp(scale)
        scale = torch.ldexp(torch.ones_like(scale), exponent - (mantissa == 0.5).int())
    codes = (v / scale).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(tokens, -1)[:, :dim].contiguous()
    return (codes, scale.squeeze(-1)) + (() if s["residual"] is None else (h,))


def _values(codes, scales, high):
    """What codes with a scale for each ``high`` rows by 128 columns stand for, 32 bits."""
    wide = scales.repeat_interleave(high, 0)[:codes.shape[0]].repeat_interleave(BLOCK, 1)[:, :codes.shape[1]]
    return codes.float() * wide


def _plain_product(s):
    return (_values(s["a"], s["a_scales"], 1) @ _values(s["b"], s["b_scales"], BLOCK).t()).to(s["dtype"])


def _plain_ancestors(s):
    """Whether drafted token j is t or an ancestor of it, and how many there are above t."""
    parents = s["parents"].long()
    batch, drafts = parents.shape
    token = torch.arange(drafts, device=DEVICE)
    there = (parents >= -1) & (parents < token)
    seen = torch.zeros((batch, drafts, drafts), device=DEVICE, dtype=torch.bool)
    at, alive = token.expand(batch, -1), there
    for _ in range(drafts):  # one generation up at a time
        seen |= alive[..., None] & (at[..., None] == token)
        up = parents.gather(1, at.clamp_min(0))
        alive = alive & (up >= 0)
        at = torch.where(alive, up, 0)
    return seen, (seen.sum(-1) - 1).clamp_min(0), there


def _packed(seen):
    """32 truth values a word, the first in the lowest bit."""
    words = -(-seen.shape[-1] // 32)
    bits = torch.nn.functional.pad(seen.long(), (0, words * 32 - seen.shape[-1])).unflatten(-1, (words, 32))
    value = (bits << torch.arange(32, device=seen.device)).sum(-1)
    return torch.where(value >= 1 << 31, value - (1 << 32), value).int()


def _rows(s, flat):
    """Cache rows [n, 576] of the flat row numbers, 32 bits."""
    kv = s["kv"].view(-1, s["kv"].shape[-1])[flat]
    if s["k_rope"] is not None:
        return torch.cat([kv, s["k_rope"].view(-1, ROPE)[flat]], -1).float()
    codes = kv[..., :LATENT].contiguous().view(torch.float8_e4m3fn).float()
    scale = kv[..., LATENT:LATENT + 16].contiguous().view(torch.float32)
    latent = (codes.unflatten(-1, (4, 128)) * scale[..., None]).flatten(-2)
    return torch.cat([latent, kv[..., LATENT + 16:].contiguous().view(torch.bfloat16).float()], -1)


def _plain_tree(s):
    batch, drafts, heads, _ = s["q"].shape
    prefix, table, lengths = s["prefix"], s["block_table"], s["lengths"].long()
    seen, depth, there = _plain_ancestors(s)
    if table is None:
        total = s["kv"].shape[1]
        flat = torch.arange(batch * total, device=DEVICE).view(batch, total)
    else:
        block = s["kv"].shape[1]
        flat = (table.long()[:, :, None] * block + torch.arange(block, device=DEVICE)).flatten(1)
        total = flat.shape[1]
    key = torch.arange(total, device=DEVICE)
    behind = key - lengths[:, None]
    drafted = seen.gather(2, behind.clamp(0, drafts - 1)[:, None].expand(-1, drafts, -1))
    visible = (behind < 0)[:, None] | (((behind >= 0) & (behind < drafts))[:, None] & drafted)
    flat[:, :prefix] = flat[0, :prefix].clone()
    out = torch.empty((batch, drafts, heads, LATENT), device=DEVICE, dtype=torch.bfloat16)
    peak = torch.empty((batch, 1, drafts, heads), device=DEVICE)
    norm = torch.empty_like(peak)
    q = torch.cat([s["q"], s["q_rope"]], -1).float().view(batch, drafts * heads, WIDTH)
    for b in range(batch):
        rows = _rows(s, flat[b])
        score = (q[b] @ rows.t()).view(drafts, heads, total) * (DEFAULT_SCALE if s["scale"] is None else s["scale"])
        score = score.masked_fill(~visible[b][:, None], -math.inf)
        top = score.amax(-1, keepdim=True)
        weight = torch.exp(score - top.clamp_min(torch.finfo(torch.float32).min))
        sums = weight.sum(-1, keepdim=True)
        weight = (weight / torch.where(sums > 0, sums, 1.0)).view(drafts * heads, total)
        out[b] = (weight @ rows[:, :LATENT]).view(drafts, heads, LATENT)
        peak[b, 0], norm[b, 0] = top[..., 0], sums[..., 0]
    return _packed(seen), torch.where(there, lengths[:, None] + depth, 0).int(), out, peak, norm


# ------------------------------------------------------------------ one pass

def run(state):
    op = state["op"]
    if not own:
        plain = {"norm": _plain_norm, "codes": _plain_codes, "product": _plain_product, "tree": _plain_tree}
        return plain[op](state)
    import dsa_amd

    s = state
    if op == "norm":
        if not s["grad"]:
            out = dsa_amd.rms_norm(s["x"], s["weight"], s["residual"], eps=EPS)
            return out if type(out) is tuple else (out,)
        out = dsa_amd.rms_norm(s["x"], s["weight"], s["residual"], eps=EPS)
        out = out if type(out) is tuple else (out,)
        leaves = [t for t in (s["x"], s["residual"], s["weight"]) if t is not None]
        return (*(t.detach() for t in out), *torch.autograd.grad(out, leaves, s["given"]))
    if op == "codes":
        if s["weight"] is None:
            return dsa_amd.quantize_fp8(s["x"], pow2_scales=s["pow2"])
        return dsa_amd.rms_norm_fp8(s["x"], s["weight"], s["residual"], eps=EPS, pow2_scales=s["pow2"])
    if op == "product":
        return dsa_amd.matmul_fp8(s["a"], s["a_scales"], s["b"], s["b_scales"], dtype=s["dtype"])
    tree, positions = dsa_amd.draft_tree(s["parents"], s["lengths"])
    return (tree, positions, *dsa_amd.forward_tree(s["q"], s["kv"], s["q_rope"], s["k_rope"], s["lengths"], tree,
                                                   s["prefix"], scale=s["scale"], block_table=s["block_table"]))


# ------------------------------------------------------------------ bounds

def work(case):
    """Bytes and operations of one pass: each input read once, each output written once."""
    op = case["op"]
    if op == "norm":
        size = 4 if case["dtype"] == "f32" else 2
        values = case["tokens"] * case["dim"]
        streams = 4 if case["residual"] else 2  # x, y and with a residual that and the sum
        if case["grad"]:
            streams += 3 if case["residual"] else 2  # the given gradients, the stream's
        return {"bytes": size * (streams * values + (2 if case["grad"] else 1) * case["dim"]),
                "flops": values * (14 if case["grad"] else 5)}
    if op == "codes":
        values = case["tokens"] * case["dim"]
        return {"bytes": values * (2 + 1 + (4 if case["residual"] else 0)) + 4 * case["tokens"] * -(-case["dim"] // BLOCK)
                + (2 * case["dim"] if case["norm"] else 0),
                "flops": values * (8 if case["norm"] else 3)}
    if op == "product":
        rows, cols, inner = case["rows"], case["cols"], case["inner"]
        blocks = -(-inner // BLOCK)
        return {"bytes": (rows + cols) * inner + 4 * blocks * (rows + -(-cols // BLOCK))
                + rows * cols * (4 if case["dtype"] == "f32" else 2),
                "flops": 2 * rows * cols * inner}
    live = case["batch"] - (1 if case["padded"] else 0)
    prefix = case["prefix"]
    own_rows = case["context"] - prefix - ((case["context"] - prefix) // 4 if case["ragged"] else 0)
    rows = live * case["drafts"] * case["heads"]
    cached = prefix + live * (own_rows + case["drafts"])
    return {"bytes": (cached * (FP8_ROW if case["cache"] == "fp8" else 2 * WIDTH)
                      + case["batch"] * case["drafts"] * case["heads"] * (2 * WIDTH + 2 * LATENT + 8)),
            "flops": 2 * rows * (prefix + own_rows) * (WIDTH + LATENT)}


# ------------------------------------------------------------------ 64 bits

def _exact_stream(s):
    """The sum in 64 bits, and what the norm is taken of: the sum as the stream keeps it."""
    x = s["x"].detach()
    if s["residual"] is None:
        return None, x.double()
    total = x.double() + s["residual"].detach().double()
    return total, total.to(x.dtype).double()


def _exact_norm(s):
    total, h = _exact_stream(s)
    weight = s["weight"].detach().double()
    size = (h.square().sum(-1) / h.shape[1] + EPS).sqrt()[:, None]
    outputs = [weight * h / size] + ([] if total is None else [total])
    if s["grad"]:
        back = s["given"][0].double() * weight
        # d(h / size) = dh / size - h (h . dh) / (n size^3)
        dx = back / size - h * ((h * back).sum(-1, keepdim=True) / (h.shape[1] * size ** 3))
        if total is not None:
            dx += s["given"][1].double()
        outputs += [dx] + ([] if total is None else [dx]) + [(s["given"][0].double() * h / size).sum(0)]
    return tuple(outputs)


def _exact_codes(s):
    total, v = _exact_stream(s)
    if s["weight"] is not None:
        v = v * s["weight"].double() / (v.square().sum(-1, keepdim=True) / v.shape[1] + EPS).sqrt()
    scales, codes = [], torch.empty_like(v)
    for first in range(0, v.shape[1], BLOCK):
        part = v[:, first:first + BLOCK]
        scale = part.abs().amax(1) / E4M3_MAX
        if s["pow2"]:
            scale = torch.exp2(torch.ceil(torch.log2(scale)))
        scale = torch.where(scale > 0, scale, 1.0)
        codes[:, first:first + BLOCK] = part / scale[:, None]
        scales.append(scale)
    return (codes, torch.stack(scales, 1)) + (() if total is None else (total,))


def _exact_product(s):
    """Block after block of the inner dimension."""
    a, b = s["a"], s["b"]
    out = torch.zeros((a.shape[0], b.shape[0]), device=DEVICE, dtype=torch.float64)
    band = torch.arange(b.shape[0], device=DEVICE) // BLOCK
    for k in range(s["a_scales"].shape[1]):
        part = slice(k * BLOCK, (k + 1) * BLOCK)
        left = a[:, part].double() * s["a_scales"][:, k, None].double()
        right = b[:, part].double() * s["b_scales"][band, k, None].double()
        out += left @ right.t()
    return out


def _exact_tree(s):
    """Sequence by sequence; the ancestors on the host, token by token."""
    batch, drafts, heads, _ = s["q"].shape
    scale = DEFAULT_SCALE if s["scale"] is None else s["scale"]
    words = -(-drafts // 32)
    masks, positions = [], []
    for row, held in zip(s["parents"].tolist(), s["lengths"].tolist()):
        bits, place = [], []
        for t, parent in enumerate(row):
            if parent < -1 or parent >= t or (parent >= 0 and bits[parent] == 0):
                bits.append(0)
                place.append(0)
            else:
                bits.append(1 << t | (bits[parent] if parent >= 0 else 0))
                place.append(place[parent] + 1 if parent >= 0 else held)
        masks.append(bits)
        positions.append(place)
    packed = [[[(m >> 32 * w & 0xffffffff) - (m >> (32 * w + 31) & 1) * (1 << 32) for w in range(words)] for m in bits]
              for bits in masks]
    out = torch.zeros((batch, drafts, heads, LATENT), device=DEVICE, dtype=torch.float64)
    peak = torch.full((batch, 1, drafts, heads), -math.inf, device=DEVICE, dtype=torch.float64)
    total = torch.zeros_like(peak)
    for b, held in enumerate(s["lengths"].tolist()):
        key = torch.arange(held + drafts, device=DEVICE)
        sequence = torch.where(key < s["prefix"], 0, b)
        if s["block_table"] is None:
            flat = sequence * s["kv"].shape[1] + key
        else:
            block = s["kv"].shape[1]
            flat = s["block_table"].long()[sequence, key // block] * block + key % block
        rows = _rows(s, flat).double()
        seen = torch.tensor([[m >> j & 1 for j in range(drafts)] for m in masks[b]], device=DEVICE, dtype=torch.bool)
        step = max(1, (1 << 27) // (heads * (held + drafts)))
        for i in range(0, drafts, step):
            q = torch.cat([s["q"][b, i:i + step], s["q_rope"][b, i:i + step]], -1).double()
            score = (q.flatten(0, 1) @ rows.t()).view(q.shape[0], heads, -1) * scale
            score[..., held:].masked_fill_(~seen[i:i + step, None], -math.inf)
            top = score.amax(-1)
            live = top > -math.inf
            weight = torch.exp(score - torch.where(live, top, 0.0)[..., None])
            norm = weight.sum(-1)
            latent = (weight.flatten(0, 1) @ rows[:, :LATENT]).view(q.shape[0], heads, LATENT)
            out[b, i:i + step] = latent / torch.where(live, norm, 1.0)[..., None]
            peak[b, 0, i:i + step], total[b, 0, i:i + step] = top, norm
    return (torch.tensor(packed, dtype=torch.int32), torch.tensor(positions, dtype=torch.int32), out, peak, total)


def exact(case, seed):
    s = prepare(case, seed)
    compute = {"norm": _exact_norm, "codes": _exact_codes, "product": _exact_product, "tree": _exact_tree}
    return compute[case["op"]](s)
