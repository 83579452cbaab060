"""The rotary, windowed attention and 4-bit operators as they are used together: a decoder layer over a
cache, prompt at once and then token by token; and the engine with its adaLN cores in 4 bits."""

import pytest
import torch

from iris_mi355x import kernels as K
from iris_mi355x import tables
from iris_mi355x.config import RELEASED_TOPOLOGY
from iris_mi355x.engine import HipIris
from iris_mi355x.weights import synthetic_state_dict
from oracle import iris_oracle as O
from parity import check

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16
WIDTH, HEADS, KV, HD, ROWS = 256, 4, 2, 128, 96


def dense(codes, scales):
    w = torch.stack([codes & 15, codes >> 4], -1).flatten(1).double() - 8
    of = torch.arange(w.shape[1], device=codes.device) // 64
    return w * scales.double()[:, of]


class Layer:
    """Projection, rotary, cache, windowed attention, output projection of ``B`` sequences."""

    def __init__(self, batch, window, sinks, seed=0):
        g = torch.Generator(device=DEV).manual_seed(seed)
        width = (HEADS + 2 * KV) * HD
        self.qkv = K.pack_w4(torch.randn(width, WIDTH, generator=g, device=DEV) * WIDTH ** -0.5)[:2]
        self.proj = K.pack_w4(torch.randn(WIDTH, HEADS * HD, generator=g, device=DEV) * (HEADS * HD) ** -0.5)[:2]
        self.freqs, self.factor = tables.rotary_frequencies(64, 10000.0, DEV, "by_parts", 4.0, trained=32)
        self.window, self.sinks = window, sinks
        self.caches = [torch.full((batch, KV, ROWS, HD), float("nan"), device=DEV, dtype=BF16) for _ in range(2)]
        self.lengths = torch.zeros(batch, device=DEV, dtype=torch.int64)

    def heads(self, x):
        """``[B, N, WIDTH]`` FP32 -> q, k, v views of the BF16 projection."""
        batch, n, _ = x.shape
        p = torch.empty(batch * n, (HEADS + 2 * KV) * HD, device=DEV, dtype=BF16)
        K.gemv_w4(*self.qkv, x.reshape(batch * n, WIDTH), None, p)
        p = p.view(batch, n, HEADS + 2 * KV, HD)
        return p[:, :, :HEADS], p[:, :, HEADS:HEADS + KV], p[:, :, HEADS + KV:]

    def step(self, x, rows, lengths):
        """Tokens ``x`` at cache rows ``rows`` ``[B, N]`` (-1: padding); ``lengths`` after them."""
        q, k, v = self.heads(x)
        q = K.rotary_store(q, k, v, rows, self.freqs, *self.caches, factor=self.factor, layout="interleaved")
        o = K.window_attention(q, *self.caches, self.window, self.sinks, lengths=lengths, starts=rows[:, 0].contiguous())
        out = torch.empty(o.shape[0] * o.shape[1], WIDTH, device=DEV)
        K.gemv_w4(*self.proj, o.view(-1, HEADS * HD), None, out)
        return out.view(*x.shape)

    def reference(self, x, n):
        """The layer over the first ``n`` tokens of one item, FP64, at the BF16 points of the operators."""
        p = (x[:n].double() @ dense(*self.qkv).T).to(BF16).double().view(n, HEADS + 2 * KV, HD)
        ang = torch.arange(n, device=DEV).double()[:, None, None] * self.freqs
        c, s = self.factor * ang.cos(), self.factor * ang.sin()
        turned = p[:, :HEADS + KV].clone()
        a, b = p[:, :HEADS + KV, 0:64:2], p[:, :HEADS + KV, 1:64:2]
        turned[..., 0:64:2], turned[..., 1:64:2] = a * c - b * s, b * c + a * s
        turned = turned.to(BF16).double()
        q = turned[:, :HEADS].transpose(0, 1)
        k, v = (t.transpose(0, 1).repeat_interleave(HEADS // KV, 0) for t in (turned[:, HEADS:], p[:, HEADS + KV:]))
        i, j = torch.arange(n, device=DEV)[:, None], torch.arange(n, device=DEV)
        seen = (j <= i) & ((i - j < self.window) | (j < self.sinks))
        w = torch.softmax((q @ k.transpose(1, 2) * HD ** -0.5).masked_fill(~seen, -torch.inf), -1)
        o = (w @ v).transpose(0, 1).reshape(n, HEADS * HD).to(BF16).double()
        return o @ dense(*self.proj).T


def assert_near(got, want):
    """BF16 steps of the projection and of the rotated heads that fall the other way (an FP32 sum beside a
    rounding border) reach the scores and values by 2^-8 of their size, P and the output rows are rounded by up
    to 2^-8: four such steps of the output's size at the most, in norm; and four times that in one element."""
    err = (got.double() - want)
    scale = want.norm() / want.numel() ** 0.5
    assert err.norm() <= 4 * 2.0 ** -8 * want.norm()
    assert err.abs().max() <= 16 * 2.0 ** -8 * max(scale.item(), want.abs().max().item())


def test_prompt_then_tokens():
    """Two ragged prompts, right-padded, then tokens one by one, against the whole layer; the cache's other
    rows hold NaN throughout."""
    g = torch.Generator(device=DEV).manual_seed(1)
    layer = Layer(2, window=20, sinks=3)
    x = torch.randn(2, 60, WIDTH, generator=g, device=DEV)
    first = [40, 33]
    n = max(first)
    rows = torch.arange(n, device=DEV).expand(2, -1).contiguous()
    for b in range(2):
        rows[b, first[b]:] = -1
    lengths = torch.tensor(first, device=DEV)
    got = layer.step(x[:, :n], rows, lengths)
    for b in range(2):
        assert_near(got[b, :first[b]], layer.reference(x[b], first[b]))
        assert torch.isnan(layer.caches[0][b, :, first[b]:]).all()  # padding went nowhere
    for step in range(15):
        at = torch.tensor([[first[0] + step], [first[1] + step]], device=DEV)
        lengths = lengths + 1
        token = torch.stack([x[b, at[b, 0]] for b in range(2)])[:, None]
        got = layer.step(token, at, lengths)
        for b in range(2):
            want = layer.reference(x[b], int(lengths[b]))[-1]
            assert_near(got[b, 0], want)


def test_captured_token_step():
    """One captured step, replayed over growing caches, each replay against the eager call."""
    g = torch.Generator(device=DEV).manual_seed(2)
    layer, eager = Layer(2, 16, 2), Layer(2, 16, 2)
    for one in (layer, eager):
        one.caches = [torch.zeros_like(c) for c in one.caches]
    x = torch.randn(2, 1, WIDTH, generator=g, device=DEV)
    rows = torch.zeros(2, 1, device=DEV, dtype=torch.int64)
    lengths = torch.ones(2, device=DEV, dtype=torch.int64)
    layer.step(x, rows, lengths)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer.step(x, rows, lengths)
    for step in range(30):
        x.normal_(generator=g)
        rows.fill_(step)
        lengths.fill_(step + 1)
        graph.replay()
        assert torch.equal(out, eager.step(x, rows, lengths))
        assert all(torch.equal(a, b) for a, b in zip(layer.caches, eager.caches))


@pytest.mark.parametrize("graphs", [True, False])
def test_engine_with_cores_in_four_bits(graphs):
    """The engine with ``core_bits=4`` against the oracle over the rounded cores; and the rounding shows."""
    cfg = RELEASED_TOPOLOGY
    sd = synthetic_state_dict(cfg)
    rounded = dict(sd)
    for name in ("modulation_cores.adaln_img.weight", "modulation_cores.adaln_txt.weight"):
        rounded[name] = dense(*K.pack_w4(sd[name])[:2]).to(sd[name].dtype)
    engine = HipIris(cfg, sd, device=DEV, core_bits=4, graphs=graphs)
    g = torch.Generator().manual_seed(3)
    x, t = torch.randn(2, 3, 32, 48, generator=g), torch.tensor([125.0, 850.0])
    text = torch.randn(2, cfg.text_len, cfg.hidden_size, generator=g)
    want = O.forward(rounded, cfg, x, t, prepared_text=text)
    args = [a.to(DEV) for a in (x, t, text)]
    got = engine(*args)
    check(got, want, "adaLN cores in 4 bits")
    assert torch.equal(engine(*args), got)  # deterministic, the replayed graph as the first call
    assert not torch.equal(got, HipIris(cfg, sd, device=DEV)(*args))


def test_engine_refuses_other_core_bits():
    with pytest.raises(ValueError, match="core_bits"):
        HipIris(RELEASED_TOPOLOGY, {}, device=DEV, core_bits=8)
