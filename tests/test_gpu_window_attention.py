"""``window_attention`` against FP64: windows, first visible keys, ragged lengths, masks, grouped heads,
strides, long caches, empty rows and non-finite values in places that a query does not see."""

import pytest
import torch

from iris_mi355x import kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


def visible(batch, nq, nk, window, sinks, causal, lengths, starts, key_mask):
    j = torch.arange(nk, device=DEV)
    length = torch.full((batch,), nk, device=DEV) if lengths is None else lengths.long().clamp(0, nk)
    if starts is None:
        start = length - nq
    else:
        start = starts.long() if isinstance(starts, torch.Tensor) else torch.full((batch,), starts, device=DEV)
    p = start[:, None, None] + torch.arange(nq, device=DEV)[:, None]
    seen = (j < length[:, None, None]).expand(batch, nq, nk)
    if causal:
        seen = seen & (j <= p)
    if window is not None:
        seen = seen & (((p - j).abs() < window) | (j < sinks))
    if key_mask is not None:
        seen = seen & (key_mask != 0)[:, None, :]
    return seen


def reference(q, k, v, window=None, sinks=0, causal=True, lengths=None, starts=None, key_mask=None, scale=None):
    """``(o, tolerance)`` in FP64, ``[B, Nq, H, 128]``.

    The kernel's scores are FP32 sums of 128 exact products (128 2^-24 of their absolute sum at worst), its
    weights carry the exponential's and the sum's FP32 errors (n_k 2^-24 at worst) and are rounded to BF16
    (half a step, 2^-8) before the product with v; the result is rounded to BF16 once more."""
    group = q.shape[1] // k.shape[1]
    scale = 128 ** -0.5 if scale is None else scale
    seen = visible(q.shape[0], q.shape[2], k.shape[2], window, sinks, causal, lengths, starts, key_mask)[:, None]
    kd, vd = (t.double().repeat_interleave(group, 1) for t in (k, v))
    # hidden places count for nothing, whatever they hold
    some = seen.any(2)[:, :, :, None]
    kd, vd = torch.where(some, kd, 0.0), torch.where(some, vd, 0.0)
    s = (q.double() @ kd.transpose(-1, -2) * scale).masked_fill(~seen, -torch.inf)
    off = (q.double().abs() @ kd.abs().transpose(-1, -2) * abs(scale) * 128 * 2.0 ** -24).masked_fill(~seen, 0.0).amax(-1, True)
    w = torch.where(seen.any(-1, True), torch.softmax(s, -1), 0.0)
    o, a = w @ vd, w @ vd.abs()
    tol = (2.0 ** -8 + 2 * off + (k.shape[2] + 16) * 2.0 ** -24) * a + 2.0 ** -8 * o.abs() * 1.01 + 1e-30
    return o.transpose(1, 2), tol.transpose(1, 2)


def check(q, k, v, got=None, **options):
    if got is None:
        got = K.window_attention(q, k, v, **options)
    options.pop("out", None)
    want, tol = reference(q, k, v, **options)
    assert got.shape == (q.shape[0], q.shape[2], q.shape[1] * 128) and got.dtype == BF16
    err = (got.unflatten(-1, (-1, 128)).double() - want).abs()
    assert (err <= tol).all(), f"worst {(err / tol.clamp(min=1e-30)).max().item():.3g} of the tolerance"


def heads_of(seed, batch, nq, nk, heads, kv, gain=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    q = gain * torch.randn(batch, heads, nq, 128, generator=g, device=DEV)
    k, v = (torch.randn(batch, kv, nk, 128, generator=g, device=DEV) for _ in range(2))
    return q.to(BF16), k.to(BF16), v.to(BF16)


@pytest.mark.parametrize("n", [1, 2, 31, 33, 64, 65, 127, 128, 200, 300, 513])
@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (7, 1), (64, 4), (100, 70), (128, 0), (1000, 3)])
@pytest.mark.parametrize("causal", [True, False])
def test_prompts(n, window, sinks, causal):
    q, k, v = heads_of(20, 2, n, n, 4, 1, gain=2.0)
    check(q, k, v, window=window, sinks=sinks, causal=causal)


@pytest.mark.parametrize("heads,kv", [(1, 1), (2, 2), (6, 2), (5, 1), (20, 5), (8, 1), (21, 3), (16, 1), (32, 1)])
@pytest.mark.parametrize("nq,nk", [(1, 77), (3, 1000), (150, 150), (17, 400)])
def test_grouped_heads(heads, kv, nq, nk):
    q, k, v = heads_of(21, 2, nq, nk, heads, kv)
    check(q, k, v, window=50, sinks=3)
    check(q, k, v)


@pytest.mark.parametrize("nq", [1, 2, 4, 5, 16, 33])
@pytest.mark.parametrize("nk", [40, 64, 1000, 4097])
@pytest.mark.parametrize("window,sinks", [(None, 0), (256, 4), (1, 0), (3000, 130)])
def test_few_queries_over_a_cache(nq, nk, window, sinks):
    q, k, v = heads_of(22, 3, nq, nk, 20, 5)
    lengths = torch.tensor([nk, max(nq, nk // 2), min(nq, nk)], device=DEV, dtype=torch.int32)
    check(q, k, v, window=window, sinks=sinks)
    check(q, k, v, window=window, sinks=sinks, lengths=lengths)
    check(q, k, v, window=window, sinks=sinks, lengths=lengths.long(), causal=False)


@pytest.mark.parametrize("nk", [16385, 40000])
@pytest.mark.parametrize("batch", [1, 7])
def test_long_caches(nk, batch):
    q, k, v = heads_of(23, batch, 1, nk, 8, 2, gain=3.0)
    lengths = torch.arange(batch, device=DEV) * (nk // 9) + nk // 3
    check(q, k, v)
    check(q, k, v, lengths=lengths)
    check(q, k, v, lengths=lengths, window=nk // 2, sinks=100)


def test_one_query_of_a_peaked_row():
    """One key far above the others, in the last place, the first, and beside the window's edge."""
    for at in (0, 1, 499, 500, 998, 999):
        q, k, v = heads_of(24, 1, 1, 1000, 4, 1)
        k[0, 0, at] = 4 * q[0, 0, 0]
        check(q, k, v)
        check(q, k, v, window=500, sinks=1)


@pytest.mark.parametrize("nq,nk", [(1, 300), (120, 120), (130, 700)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("kind", [torch.bool, torch.uint8])
def test_key_masks(nq, nk, causal, kind):
    q, k, v = heads_of(25, 4, nq, nk, 4, 2)
    g = torch.Generator(device=DEV).manual_seed(1)
    mask = (torch.rand(4, nk, generator=g, device=DEV) < 0.6)
    mask[1, : nk // 2] = False  # padding in front
    mask[2] = False  # nothing at all
    mask = mask.to(kind) * (3 if kind == torch.uint8 else 1)
    mask = mask.to(kind)
    for window, sinks in ((None, 0), (20, 2), (90, 0)):
        out = torch.full((4, nq, 512), 7.0, device=DEV, dtype=BF16)
        got = K.window_attention(q, k, v, window, sinks, causal=causal, key_mask=mask, out=out)
        assert got is out and not got[2].any()
        check(q, k, v, got, window=window, sinks=sinks, causal=causal, key_mask=mask)


@pytest.mark.parametrize("starts", [0, 5, -3, 1000, 10**12, "ints"])
@pytest.mark.parametrize("nq,nk", [(1, 64), (40, 200), (200, 200)])
@pytest.mark.parametrize("causal", [True, False])
def test_starts(starts, nq, nk, causal):
    """Right-padded prompts (starts 0, lengths below Nq), queries before the first key and far past the last."""
    q, k, v = heads_of(26, 3, nq, nk, 4, 2)
    if starts == "ints":
        starts = torch.tensor([0, nk // 2, -nq], device=DEV)
    lengths = torch.tensor([nk, nk // 3, 0], device=DEV)
    for window, sinks in ((None, 0), (33, 2), (2 * 10**12, 0)):
        check(q, k, v, window=window, sinks=sinks, causal=causal, lengths=lengths, starts=starts)


def test_lengths_are_clamped():
    q, k, v = heads_of(27, 3, 2, 50, 2, 1)
    lengths = torch.tensor([-4, 60, 2**40], device=DEV)
    got = K.window_attention(q, k, v, lengths=lengths)
    assert not got[0].any()
    check(q, k, v, got, lengths=lengths)


@pytest.mark.parametrize("nq,nk", [(1, 500), (130, 130)])
def test_strided_views(nq, nk):
    """Token-major and packed views, an expanded batch of keys, an output with room between rows."""
    g = torch.Generator(device=DEV).manual_seed(28)
    q = torch.randn(3, nq, 8, 136, generator=g, device=DEV).to(BF16)[..., :128].transpose(1, 2)
    packed = torch.randn(1, nk, 5, 128, generator=g, device=DEV).to(BF16)
    k, v = packed[:, :, 0:2].transpose(1, 2).expand(3, -1, -1, -1), packed[:, :, 3:5].transpose(1, 2).expand(3, -1, -1, -1)
    store = torch.full((3, nq + 2, 1100), 7.0, device=DEV, dtype=BF16)
    out = store[:, 1:-1, 4:1028]
    K.window_attention(q, k, v, 60, 2, out=out)
    check(q, k, v, out, window=60, sinks=2)
    store[:, 1:-1, 4:1028] = 7.0
    assert (store == 7.0).all()


def test_offsets_past_32_bits():
    rows, stride = 40, 1 << 26
    flat = torch.empty(rows * stride, device=DEV, dtype=BF16)
    k = flat.as_strided((1, 1, rows, 128), (rows * stride, 128, stride, 1))
    v = flat.as_strided((1, 1, rows, 128), (rows * stride, 128, stride, 1), 256)
    g = torch.Generator(device=DEV).manual_seed(29)
    k.copy_(torch.randn(rows, 128, generator=g, device=DEV))
    v.copy_(torch.randn(rows, 128, generator=g, device=DEV))
    for nq in (1, 40):
        q = torch.randn(1, 4, nq, 128, generator=g, device=DEV).to(BF16)
        got = K.window_attention(q, k, v, 30, 2)
        check(q, k.contiguous(), v.contiguous(), got, window=30, sinks=2)


@pytest.mark.parametrize("nq,nk,causal", [(1, 400, True), (3, 400, True), (200, 200, True), (200, 200, False)])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_non_finite_values_in_hidden_places(nq, nk, causal, value):
    """Masked keys, keys past the length and keys outside every query's window hold NaN or infinities; and one
    key that later queries see does: the rows before it, and after its window, are as if it were not there."""
    q, k, v = heads_of(30, 2, nq, nk, 4, 2)
    mask = torch.ones(2, nk, device=DEV, dtype=torch.bool)
    mask[0, 5:9], mask[1, nk - 40: nk - 35] = False, False
    lengths = torch.tensor([nk, nk - 3], device=DEV)
    for window, sinks in ((None, 0), (60, 2)):
        seen = visible(2, nq, nk, window, sinks, causal, lengths, None, mask)
        kb, vb = k.clone(), v.clone()
        hidden = ~seen.any(1)[:, None, :, None]
        kb.masked_fill_(hidden, value), vb.masked_fill_(hidden, value)
        options = dict(window=window, sinks=sinks, causal=causal, key_mask=mask, lengths=lengths)
        got = K.window_attention(q, kb, vb, **options)
        check(q, k, v, got, **options)
        at = nk - 30
        kb, vb = k.clone(), v.clone()
        vb[:, :, at, 3] = value
        got = K.window_attention(q, kb, vb, **options).unflatten(-1, (-1, 128))
        touched = torch.zeros_like(got, dtype=torch.bool)
        touched[..., 3] = seen[:, :, at, None]
        assert not torch.isfinite(got[touched]).any()
        want, tol = reference(q, k, v, **options)
        assert ((got.double() - want).abs() <= tol)[~touched].all()
        kb[:, :, at, 7], vb = value, v
        got = K.window_attention(q, kb, vb, **options).unflatten(-1, (-1, 128))
        assert ((got.double() - want).abs() <= tol)[~seen[:, :, at]].all()


def test_rows_do_not_depend_on_the_batch():
    q, k, v = heads_of(31, 4, 1, 5000, 8, 2)
    whole = K.window_attention(q, k, v, 2000, 4)
    for b in range(4):
        one = K.window_attention(q[b:b + 1], k[b:b + 1], v[b:b + 1], 2000, 4)
        assert torch.allclose(one.double(), whole[b:b + 1].double(), rtol=2.0 ** -7, atol=2.0 ** -8)
    assert torch.equal(whole, K.window_attention(q, k, v, 2000, 4))  # and not on the run


def test_empty_calls():
    for batch, nq, nk in ((0, 3, 5), (2, 0, 5), (2, 3, 0)):
        q, k, v = heads_of(32, batch, nq, nk, 2, 1)
        got = K.window_attention(q, k, v, 4, 1)
        assert got.shape == (batch, nq, 256) and not got.any()


def test_streams_and_graphs():
    """Two captured graphs of split calls replayed in turns, on another stream, with eager calls between."""
    q, k, v = heads_of(33, 2, 1, 9000, 8, 2)
    outs = [torch.empty(2, 1, 1024, device=DEV, dtype=BF16) for _ in range(2)]
    lengths = torch.tensor([9000, 9000], device=DEV)
    options = [dict(lengths=lengths), dict(lengths=lengths, window=3000, sinks=4)]
    K.window_attention(q, k, v, out=outs[0], **options[0])
    torch.cuda.synchronize()
    graphs = []
    for out, opt in zip(outs, options):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            K.window_attention(q, k, v, out=out, **opt)
        graphs.append(graph)
    g = torch.Generator(device=DEV).manual_seed(3)
    side = torch.cuda.Stream()
    for step in range(3):
        q.normal_(generator=g)
        lengths.copy_(torch.tensor([9000 - 700 * step, 17 + step]))
        for graph, out, opt in zip(graphs, outs, options):
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                graph.replay()
            torch.cuda.current_stream().wait_stream(side)
            assert torch.equal(out, K.window_attention(q, k, v, **opt))


@pytest.mark.parametrize("nq", [1, 40])
def test_strides_of_axes_of_one_say_nothing(nq):
    """One item, one K/V head, one key: the strides of such axes are never taken, whatever they are."""
    q, k, v = heads_of(35, 1, nq, 70, 2, 1)
    want = K.window_attention(q, k, v, window=9)
    odd = [t.as_strided(t.shape, (12345, 777 if t.shape[1] == 1 else t.stride(1), *t.stride()[2:])) for t in (q, k, v)]
    assert torch.equal(K.window_attention(*odd, window=9), want)
    one = [t[:, :, :1].as_strided((1, 1, 1, 128), (3, 5, s, 1)) for t, s in ((k, 7), (v, 1 << 30))]
    got = K.window_attention(q, *one, causal=False)
    assert torch.equal(got.unflatten(-1, (2, 128)), v[:, :, :1].expand(1, nq, 2, 128))


def test_key_mask_shared_by_the_items():
    q, k, v = heads_of(36, 3, 100, 100, 4, 1)
    mask = torch.rand(1, 100, generator=torch.Generator().manual_seed(5)).to(DEV) < 0.6
    check(q, k, v, key_mask=mask.expand(3, -1), window=40, sinks=2)
    check(q[:, :, -1:], k, v, key_mask=mask.expand(3, -1))


# Calls of more 16-row tiles than the card has CUs (and of K/V that 32-bit offsets do not span)
@pytest.mark.parametrize("n", [17, 33, 64, 65, 130, 200])
@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (7, 1), (64, 4), (100, 70), (1000, 3)])
@pytest.mark.parametrize("causal", [True, False])
def test_many_prompts(n, window, sinks, causal):
    q, k, v = heads_of(37, 20, n, n, 8, 8, gain=2.0)
    check(q, k, v, window=window, sinks=sinks, causal=causal)


@pytest.mark.parametrize("heads,kv,batch", [(20, 5, 60), (5, 5, 70), (6, 2, 150), (6, 1, 300), (32, 2, 80)])
@pytest.mark.parametrize("nq,nk", [(1, 300), (3, 77), (16, 129)])
def test_few_queries_of_many_items(heads, kv, batch, nq, nk):
    q, k, v = heads_of(38, batch, nq, nk, heads, kv)
    g = torch.Generator(device=DEV).manual_seed(39)
    lengths = torch.randint(0, nk + 1, (batch,), generator=g, device=DEV)
    mask = torch.rand(batch, nk, generator=g, device=DEV) < 0.7
    mask[1], mask[2, : nk // 2] = False, False
    check(q, k, v, lengths=lengths)
    check(q, k, v, lengths=lengths, window=50, sinks=3, key_mask=mask)
    check(q, k, v, starts=lengths.int() - 20, window=50, causal=False, key_mask=mask, scale=-0.2)


@pytest.mark.parametrize("nq", [17, 100, 256])
@pytest.mark.parametrize("nk", [300, 5000])
@pytest.mark.parametrize("window,sinks", [(None, 0), (300, 40)])
def test_some_queries_over_a_cache(nq, nk, window, sinks):
    """Several row tiles of one K/V head, their keys split."""
    for heads, kv in ((8, 1), (4, 2), (1, 1), (3, 1)):
        q, k, v = heads_of(40, 1, nq, nk, heads, kv)
        check(q, k, v, window=window, sinks=sinks)
        check(q, k, v, window=window, sinks=sinks, causal=False, starts=max(nk - 2 * nq, 0))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_non_finite_values_in_hidden_places_of_many_items(causal, value):
    batch, n = 20, 130
    q, k, v = heads_of(41, batch, n, n, 8, 8)
    mask = torch.ones(batch, n, device=DEV, dtype=torch.bool)
    mask[0, 5:9], mask[1, 90:95], mask[5] = False, False, False
    lengths = torch.full((batch,), n, device=DEV)
    lengths[1], lengths[2], lengths[3] = n - 3, 0, 1
    for window, sinks in ((None, 0), (60, 2)):
        options = dict(window=window, sinks=sinks, causal=causal, key_mask=mask, lengths=lengths)
        seen = visible(batch, n, n, window, sinks, causal, lengths, None, mask)
        hidden = ~seen.any(1)[:, None, :, None]
        check(q, k, v, K.window_attention(q, k.masked_fill(hidden, value), v.masked_fill(hidden, value), **options), **options)
        vb = v.clone()
        vb[:, :, 100, 3] = value
        got = K.window_attention(q, k, vb, **options).unflatten(-1, (-1, 128))
        touched = torch.zeros_like(got, dtype=torch.bool)
        touched[..., 3] = seen[:, :, 100, None]
        assert touched.any() and not torch.isfinite(got[touched]).any()
        want, tol = reference(q, k, v, **options)
        assert ((got.double() - want).abs() <= tol)[~touched].all()


def test_many_rows_over_keys_that_span_two_gib():
    rows, stride = 130, 9 << 20
    flat = torch.empty(rows * stride, device=DEV, dtype=BF16)
    k = flat.as_strided((1, 1, rows, 128), (rows * stride, 128, stride, 1))
    v = flat.as_strided((1, 1, rows, 128), (rows * stride, 128, stride, 1), 256)
    g = torch.Generator(device=DEV).manual_seed(42)
    k.copy_(torch.randn(rows, 128, generator=g, device=DEV))
    v.copy_(torch.randn(rows, 128, generator=g, device=DEV))
    q = torch.randn(1, 70, 100, 128, generator=g, device=DEV).to(BF16)  # 438 row tiles
    for options in (dict(window=30, sinks=2), dict(causal=False)):
        check(q, k.contiguous(), v.contiguous(), K.window_attention(q, k, v, **options), **options)


@pytest.mark.parametrize("batch,heads,kv,nq,nk,apart", [(2, 4, 2, 1, 300, 128), (2, 4, 2, 40, 300, 128), (70, 8, 8, 130, 130, 128),
                                                        (20, 8, 8, 130, 130, 128), (1, 4, 1, 1, 40, 1 << 26),
                                                        (1, 4, 1, 40, 40, 1 << 26)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (30, 2)])
def test_scores_of_minus_infinity(batch, heads, kv, nq, nk, apart, window, sinks):
    """Keys whose scores are -inf weigh nothing, the first visible one of a row and the last among them: as if masked."""
    q, k, v = heads_of(43, batch, nq, nk, heads, kv)
    q[..., 3] = q[..., 3].abs() + 0.1
    shown = torch.ones(batch, nk, device=DEV, dtype=torch.bool)
    shown[:, [0, 1, nk // 2, nk - 3]] = False
    low = k.clone()
    low[..., 3].masked_fill_(~shown[:, None], -torch.inf)
    if apart > 128:  # rows far apart
        flat = torch.empty(nk * apart, device=DEV, dtype=BF16)
        views = [flat.as_strided((1, 1, nk, 128), (nk * apart, 128, apart, 1), 256 * i) for i in range(2)]
        views[0].copy_(low), views[1].copy_(v)
        got = K.window_attention(q, *views, window, sinks)
    else:
        got = K.window_attention(q, low, v, window, sinks)
    check(q, k, v, got, window=window, sinks=sinks, key_mask=shown)


@pytest.mark.parametrize("batch,nq,strides", [(1, 5, (3, 260, 1)), (3, 1, (520, 7, 1)), (1, 1, (1, 1, 1)), (1, 600, (2, 256, 1))])
def test_output_strides_of_axes_of_one_say_nothing(batch, nq, strides):
    q, k, v = heads_of(44, batch, nq, 600, 2, 1)
    store = torch.full((nq * 260 + batch * 520,), 7.0, device=DEV, dtype=BF16)
    out = store.as_strided((batch, nq, 256), strides)
    K.window_attention(q, k, v, 50, 2, out=out)
    assert torch.equal(out, K.window_attention(q, k, v, 50, 2))
    out.fill_(7.0)
    assert (store == 7.0).all()


@pytest.mark.parametrize("nq", [1, 70])
def test_an_output_between_its_inputs_rows(nq):
    """Query, key, value and output columns of one buffer: their rows alternate and do not meet."""
    g = torch.Generator(device=DEV).manual_seed(45)
    packed = torch.randn(2, nq, 8, 128, generator=g, device=DEV).to(BF16)
    before = packed.clone().transpose(1, 2)
    q, k, v = (packed.transpose(1, 2)[:, a:b] for a, b in ((0, 2), (2, 4), (6, 8)))
    out = packed.view(2, nq, 1024)[:, :, 512:768]
    K.window_attention(q, k, v, 30, 1, out=out)
    check(before[:, 0:2], before[:, 2:4], before[:, 6:8], out, window=30, sinks=1)
    after = packed.transpose(1, 2)
    assert torch.equal(after[:, :4], before[:, :4]) and torch.equal(after[:, 6:], before[:, 6:])


def check_norm(q, k, v, got, **options):
    """``check``, and a bound on the norm of the whole error, which leaves no room for a tile of keys left out or seen twice.

    The output's rounding is at most 2^-8 of each element. The weights' are at most 2^-8 of each and independent of one
    another: their sum over the keys has a mean square of at most (2^-16 / 3) sum w^2 v^2, and over a call's rows and dims
    its norm stays below sqrt(3) times the root of that. The FP32 terms are those of ``reference``, at their worst."""
    check(q, k, v, got, **options)
    group = q.shape[1] // k.shape[1]
    scale = options.pop("scale", None)
    seen = visible(q.shape[0], q.shape[2], k.shape[2], *(options.get(name, default) for name, default in (
        ("window", None), ("sinks", 0), ("causal", True), ("lengths", None), ("starts", None), ("key_mask", None))))[:, None]
    some = seen.any(2)[:, :, :, None]
    kd, vd = (torch.where(some, t.double().repeat_interleave(group, 1), 0.0) for t in (k, v))
    s = q.double() @ kd.transpose(-1, -2) * (128 ** -0.5 if scale is None else scale)
    w = torch.where(seen.any(-1, True), torch.softmax(s.masked_fill(~seen, -torch.inf), -1), 0.0)
    o = w @ vd
    off = q.double().norm(dim=-1).max() * kd.norm(dim=-1).max() * 128 ** -0.5 * 128 * 2.0 ** -24
    bound = 2.0 ** -8 * (o.norm() + (w.square() @ vd.square()).sum().sqrt())
    bound = bound + (2 * off + (k.shape[2] + 16) * 2.0 ** -24) * (w @ vd.abs()).norm()
    err = got.unflatten(-1, (-1, 128)).double() - o.transpose(1, 2)
    assert err.norm() <= bound, f"{(err.norm() / bound).item():.3g} of the norm's bound"


# Calls of more workgroups of 32 rows a wave than seven for four CUs: a wave holds two blocks of 16 rows.
@pytest.mark.parametrize("heads,kv", [(8, 8), (16, 8), (32, 8), (5, 5), (20, 5)])
@pytest.mark.parametrize("n", [17, 31, 32, 33, 48, 64, 65, 96, 130, 200])
@pytest.mark.parametrize("causal", [True, False])
def test_two_row_blocks(heads, kv, n, causal):
    batch = 64 if kv == 8 else 100  # (at least 500 workgroups at 32 rows of a head)
    q, k, v = heads_of(46, batch, n, n, heads, kv, gain=2.0)
    g = torch.Generator(device=DEV).manual_seed(47)
    lengths = torch.randint(0, n + 1, (batch,), generator=g, device=DEV)
    mask = torch.rand(batch, n, generator=g, device=DEV) < 0.7
    mask[1], mask[2, : n // 2] = False, False
    for options in (dict(), dict(window=20, sinks=3), dict(window=1), dict(window=40, sinks=70, key_mask=mask),
                    dict(lengths=lengths, starts=0), dict(lengths=lengths, starts=lengths - 9, window=17, key_mask=mask)):
        check_norm(q, k, v, K.window_attention(q, k, v, causal=causal, **options), causal=causal, **options)


@pytest.mark.parametrize("nq,nk", [(17, 300), (40, 129), (64, 500), (130, 257)])
@pytest.mark.parametrize("heads,kv", [(8, 8), (32, 8)])
def test_two_row_blocks_over_a_cache(nq, nk, heads, kv):
    """Query blocks whose windows end in different tiles; a negative scale; a strided output."""
    q, k, v = heads_of(48, 64, nq, nk, heads, kv)
    store = torch.full((64, nq, heads * 128 + 8), 7.0, device=DEV, dtype=BF16)
    out = store[:, :, 4:-4]
    for options in (dict(), dict(window=50, sinks=5), dict(window=65, causal=False, starts=nk // 3),
                    dict(window=nk // 2, scale=-0.15, starts=-5, causal=False)):
        check_norm(q, k, v, K.window_attention(q, k, v, out=out, **options), **options)
    out.fill_(7.0)
    assert (store == 7.0).all()


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("at", [3, 20, 70, 100])
def test_non_finite_values_in_hidden_places_of_two_row_blocks(causal, value, at):
    batch, n = 64, 130
    q, k, v = heads_of(49, batch, n, n, 8, 8)
    mask = torch.ones(batch, n, device=DEV, dtype=torch.bool)
    mask[0, 5:9], mask[1, 90:95], mask[5] = False, False, False
    lengths = torch.full((batch,), n, device=DEV)
    lengths[1], lengths[2], lengths[3] = n - 3, 0, 1
    for window, sinks in ((None, 0), (60, 2)):
        options = dict(window=window, sinks=sinks, causal=causal, key_mask=mask, lengths=lengths)
        seen = visible(batch, n, n, window, sinks, causal, lengths, None, mask)
        hidden = ~seen.any(1)[:, None, :, None]
        got = K.window_attention(q, k.masked_fill(hidden, value), v.masked_fill(hidden, value), **options)
        check_norm(q, k, v, got, **options)
        vb = v.clone()
        vb[:, :, at, 3] = value
        got = K.window_attention(q, k, vb, **options).unflatten(-1, (-1, 128))
        touched = torch.zeros_like(got, dtype=torch.bool)
        touched[..., 3] = seen[:, :, at, None]
        assert touched.any() and not torch.isfinite(got[touched]).any()
        want, tol = reference(q, k, v, **options)
        assert ((got.double() - want).abs() <= tol)[~touched].all()
        kb = k.clone()
        kb[:, :, at, 7] = value
        got = K.window_attention(q, kb, v, **options).unflatten(-1, (-1, 128))
        assert ((got.double() - want).abs() <= tol)[~seen[:, :, at]].all()


@pytest.mark.parametrize("batch,nq,nk", [(1, 1, 16385), (2, 1, 40000), (7, 1, 20000), (1, 2, 40000), (1, 16, 32768), (1, 128, 16384)])
@pytest.mark.parametrize("heads,kv", [(8, 2), (20, 5)])
def test_long_caches_in_norm(batch, nq, nk, heads, kv):
    """A 32-key tile left out of 40000 keys would be 3 % of the output, three times the bound."""
    q, k, v = heads_of(50, batch, nq, nk, heads, kv)
    for options in (dict(), dict(window=nk // 2, sinks=100)):
        check_norm(q, k, v, K.window_attention(q, k, v, **options), **options)


@pytest.mark.parametrize("nq,nk", [(1, 300), (3, 1000), (40, 200), (300, 300), (1000, 1000)])
def test_prompts_and_caches_in_norm(nq, nk):
    q, k, v = heads_of(51, 4, nq, nk, 20, 5, gain=1.5)
    for options in (dict(), dict(window=100, sinks=4), dict(window=33, causal=False)):
        check_norm(q, k, v, K.window_attention(q, k, v, **options), **options)
