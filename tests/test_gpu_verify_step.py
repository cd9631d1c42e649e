"""A layer's step that verifies drafted tokens, by all its operators: from the residual
stream through 8-bit projections into the cache, attention with the drafts' tree, and
back to the stream.  Each operator's result is compared, from the inputs that it had,
with its formula in 64 bits, by the checks and tolerances of its own tests."""
import pytest
import torch

import dsa_amd
from test_gpu_norm import check_codes, normed
from test_gpu_product import check as check_product
from test_gpu_tree import check as check_attention

pytestmark = pytest.mark.gpu

BF, FULL, E4M3 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
B, SQ, H, HIDDEN, RANK, BLOCK, WIDTH = 3, 6, 16, 656, 272, 16, 5
EPS = 1e-6


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")
    torch.cuda.init()


def weights(columns, inner, g):
    """Codes and the scales of blocks of 128 by 128."""
    high, wide = -(-columns // 128), -(-inner // 128)
    w = torch.zeros(high * 128, wide * 128)
    w[:columns, :inner] = torch.randn(columns, inner, generator=g) * inner ** -0.5
    w = w.view(high, 128, wide, 128)
    scale = w.abs().amax((1, 3)) / 448.0
    codes = (w / scale[:, None, :, None]).clamp(-448, 448).view(high * 128, -1)[:columns, :inner]
    return codes.to(E4M3).contiguous().cuda(), scale.contiguous().cuda()


def half(shape, g, gain=1.0):
    return (torch.randn(shape, generator=g) * gain).to(BF).cuda()


class Layer:
    def __init__(self, fp8, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.down, self.up, self.back = weights(RANK + 576, HIDDEN, g), weights(H * 192, RANK, g), weights(HIDDEN, H * 128, g)
        self.norms = [1 + half(n, g, 0.1) for n in (HIDDEN, RANK, 512, HIDDEN)]
        self.w_uk, self.w_uv = half((H, 128, 512), g, 512 ** -0.5), half((H, 128, 512), g, 512 ** -0.5)
        self.freq = dsa_amd.rotary_frequencies(64, scaling="yarn", factor=4.0).cuda()
        blocks = B * WIDTH
        kv, kr = half((blocks, BLOCK, 1, 512), g), half((blocks, BLOCK, 1, 64), g)
        self.pools = (dsa_amd.quantize_kv_fp8(kv, kr), None) if fp8 else (kv, kr)
        self.order = torch.randperm(blocks, generator=g).int().cuda()
        self.table = self.order.view(B, WIDTH).clone()

    def step(self, stream, delta, lengths, parents):
        s = {}
        s["codes"], s["scales"], s["stream"] = dsa_amd.rms_norm_fp8(delta, self.norms[0], stream, eps=EPS)
        s["low"] = dsa_amd.matmul_fp8(s["codes"], s["scales"], *self.down)
        s["latent"] = dsa_amd.rms_norm(s["low"][..., RANK:RANK + 512], self.norms[2], eps=EPS)
        s["q_codes"], s["q_scales"] = dsa_amd.rms_norm_fp8(s["low"][..., :RANK], self.norms[1], eps=EPS, pow2_scales=False)
        s["q"] = dsa_amd.matmul_fp8(s["q_codes"], s["q_scales"], *self.up).view(B, SQ, H, 192)
        s["tree"], s["positions"] = dsa_amd.draft_tree(parents, lengths)
        s["q_rope"] = dsa_amd.rotary(s["q"][..., 128:], s["positions"], self.freq)
        flat = s["q"][..., :128].reshape(B * SQ, H, 128).transpose(0, 1).float().contiguous()
        s["q_latent"] = torch.bmm(flat, self.w_uk.float()).transpose(0, 1).to(BF).reshape(B, SQ, H, 512).contiguous()
        at = lengths[:, None] + torch.arange(SQ, device="cuda").int()
        slots = self.table.gather(1, (at // BLOCK).long()) * BLOCK + at % BLOCK
        tokens = s["low"].view(B * SQ, -1)
        dsa_amd.write_kv_rows(s["latent"].view(B * SQ, 512), tokens[:, RANK + 512:], slots.view(-1), *self.pools,
                              positions=s["positions"].view(-1), frequencies=self.freq)
        s["out"], s["max"], s["sum"] = dsa_amd.forward_tree(s["q_latent"], self.pools[0], s["q_rope"], self.pools[1], lengths,
                                                            s["tree"], block_table=self.table)
        s["values"] = dsa_amd.project_uv(s["out"], self.w_uv).view(B, SQ, H * 128)
        s["o_codes"], s["o_scales"] = dsa_amd.quantize_fp8(s["values"])
        s["delta"] = dsa_amd.matmul_fp8(s["o_codes"], s["o_scales"], *self.back)
        s["next"], s["next_stream"] = dsa_amd.rms_norm(s["delta"], self.norms[3], s["stream"], eps=EPS)
        return s

    def rows(self):
        """The cache, sequence by sequence, in 64 bits."""
        kv = self.pools[0].view(-1, self.pools[0].shape[-1])
        if self.pools[1] is None:
            codes = kv[:, :512].contiguous().view(E4M3).double().unflatten(-1, (4, 128))
            latent = (codes * kv[:, 512:528].contiguous().view(FULL).double()[..., None]).flatten(-2)
            flat = torch.cat([latent, kv[:, 528:].contiguous().view(BF).double()], -1)
        else:
            flat = torch.cat([kv.double(), self.pools[1].view(-1, 64).double()], -1)
        at = (self.table.long()[:, :, None] * BLOCK + torch.arange(BLOCK, device="cuda")).flatten(1)
        return flat[at]


def inputs(seed):
    g = torch.Generator().manual_seed(seed)
    lengths = torch.randint(0, WIDTH * BLOCK - SQ + 1, (B,), generator=g).int().cuda()
    parents = torch.stack([torch.randint(-1, t, (B,), generator=g) if t else torch.full((B,), -1) for t in range(SQ)], 1)
    parents[1, SQ - 1] = -2  # padding
    return half((B, SQ, HIDDEN), g), half((B, SQ, HIDDEN), g), lengths, parents.int().cuda()


def check_norm(y, h, weight):
    want = normed(h, weight, EPS)
    assert ((y.double() - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -17) + 1e-30).all()


@pytest.mark.parametrize("fp8", [False, True])
def test_a_verify_step(fp8):
    layer = Layer(fp8)
    for seed in range(3):
        stream, delta, lengths, parents = inputs(seed)
        s = layer.step(stream, delta, lengths, parents)
        assert torch.equal(s["stream"], stream + delta)
        check_codes((s["codes"], s["scales"]), normed(s["stream"], layer.norms[0], EPS), True)
        flat = lambda *t: [x.reshape(B * SQ, -1) for x in t]  # noqa: E731
        check_product(*flat(s["low"], s["codes"], s["scales"]), *layer.down)
        check_norm(s["latent"], s["low"][..., RANK:RANK + 512], layer.norms[2])
        check_codes((s["q_codes"], s["q_scales"]), normed(s["low"][..., :RANK], layer.norms[1], EPS), False)
        check_product(*flat(s["q"], s["q_codes"], s["q_scales"]), *layer.up)
        rows = layer.rows()
        for b in range(B):  # the drafted rows stand behind each sequence
            drafted = rows[b, int(lengths[b]):int(lengths[b]) + SQ, :512]
            off = (drafted - s["latent"][b].double()).abs()
            # fp8 rows: half a step of e4m3, or of its least values under the scale of a block of 128
            most = s["latent"][b].double().abs().view(SQ, 4, 128).amax(-1).repeat_interleave(128, -1)
            assert (off <= (s["latent"][b].double().abs() * 2.0 ** -4 + most * 2.0 ** -10 / 224 if fp8 else 0)).all()
        seen = torch.zeros(B, SQ, rows.shape[1], dtype=torch.bool, device="cuda")
        for b in range(B):
            n = int(lengths[b])
            seen[b, :, :n] = True
            line = [0] * SQ
            for t, parent in enumerate(parents[b].tolist()):
                line[t] = 0 if parent < -1 else 1 << t | (line[parent] if parent >= 0 else 0)
                seen[b, t, n:n + SQ] = torch.tensor([line[t] >> j & 1 for j in range(SQ)], dtype=torch.bool, device="cuda")
        state = dict(q=s["q_latent"], q_rope=s["q_rope"], rows=rows)
        check_attention((s["out"], s["max"], s["sum"]), state, seen)
        values = torch.einsum("bthc,hdc->bthd", s["out"].double(), layer.w_uv.double())
        size = torch.einsum("bthc,hdc->bthd", s["out"].double().abs(), layer.w_uv.double().abs())
        assert ((s["values"].view(values.shape).double() - values).abs() <= 2.0 ** -8 * values.abs() + 512 * 2.0 ** -24 * size).all()
        check_codes((s["o_codes"], s["o_scales"]), s["values"].double(), True)
        check_product(*flat(s["delta"], s["o_codes"], s["o_scales"]), *layer.back)
        assert torch.equal(s["next_stream"], s["delta"] + s["stream"])
        check_norm(s["next"], s["next_stream"], layer.norms[3])


def test_a_captured_verify_step():
    """The whole step in a graph: replays with other inputs, between eager steps of a second layer like it."""
    layer, other = Layer(False), Layer(False)
    stream, delta, lengths, parents = inputs(0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s = layer.step(stream, delta, lengths, parents)
    for seed in range(4):
        for t, u in zip((stream, delta, lengths, parents), inputs(10 + seed)):
            t.copy_(u)
        graph.replay()
        want = other.step(stream, delta, lengths, parents)
        for name, t in s.items():
            bits = torch.uint8 if t.dtype == E4M3 else t.dtype
            assert torch.equal(t.view(bits), want[name].view(bits)), name
        assert torch.equal(layer.pools[0], other.pools[0])
        torch.cuda.synchronize()
