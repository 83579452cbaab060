"""``rotary`` and ``rotary_store`` against FP64: layouts, parts of a head, strides, far positions, caches."""

import math

import pytest
import torch

from iris_mi355x import kernels as K
from iris_mi355x import tables

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rotated(x, positions, freqs, layout, factor=1.0, transpose=False):
    """The rotation of ``[B, N, H, D]`` heads in FP64, as ``[B, H, N, D]``, and the bound on its error.

    The FP64 angle is reduced to a turn and rounded to FP32 (relative 2^-24 of an angle up to pi: 2^-22),
    cos and sin add a few 2^-24 and the factor and the rotation four more roundings: 2^-21 of the pair's
    magnitude; then half a step of the output type."""
    pos = positions if positions.dim() == 2 else positions[None]
    ang = pos.double()[:, :, None, None] * freqs
    c, s = factor * ang.cos(), factor * ang.sin() * (-1 if transpose else 1)
    y = x.double().clone()
    p = freqs.numel()
    i0 = torch.arange(p, device=x.device) * (1 if layout == "half" else 2)
    i1 = i0 + (p if layout == "half" else 1)
    a, b = x.double()[..., i0], x.double()[..., i1]
    y[..., i0], y[..., i1] = a * c - b * s, b * c + a * s
    tol = torch.zeros_like(y)
    tol[..., i0] = tol[..., i1] = 2.0 ** -21 * factor * (a.abs() + b.abs())
    tol[..., torch.cat([i0, i1])] += torch.finfo(x.dtype).eps / 2 * y[..., torch.cat([i0, i1])].abs()
    return y.transpose(1, 2), tol.transpose(1, 2)


def check(got, x, positions, freqs, layout, factor=1.0, transpose=False):
    want, tol = rotated(x, positions, freqs, layout, factor, transpose)
    assert got.shape == want.shape
    assert ((got.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,part", [(128, 128), (128, 64), (64, 16), (80, 40), (80, 20), (256, 256), (6, 2), (10, 10)])
def test_layouts_and_parts(dtype, layout, dim, part):
    g = torch.Generator(device=DEV).manual_seed(1)
    batch, n, heads, kv = 2, 37, 5, 1
    proj = torch.randn(batch, n, (heads + 2 * kv) * dim, generator=g, device=DEV).to(dtype)
    q = proj[..., : heads * dim].view(batch, n, heads, dim)
    k = proj[..., heads * dim: (heads + kv) * dim].view(batch, n, kv, dim)
    freqs, _ = tables.rotary_frequencies(part, 10000.0, DEV)
    positions = torch.randint(-50, 1 << 20, (batch, n), generator=g, device=DEV)
    for transpose in (False, True):
        qo, ko = K.rotary(q, k, positions, freqs, layout=layout, factor=1.25, transpose=transpose)
        check(qo, q, positions, freqs, layout, 1.25, transpose)
        check(ko, k, positions, freqs, layout, 1.25, transpose)


@pytest.mark.parametrize("batch,n,heads", [(1, 1, 1), (3, 1, 40), (1, 1000, 2), (2, 333, 7), (5, 8, 1)])
@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_sizes_and_shared_positions(batch, n, heads, kind):
    g = torch.Generator(device=DEV).manual_seed(2)
    x = torch.randn(batch, n, heads, 128, generator=g, device=DEV).to(torch.bfloat16)
    freqs, _ = tables.rotary_frequencies(128, 10000.0, DEV)
    positions = torch.arange(n, device=DEV, dtype=kind) + 70000
    got, none = K.rotary(x, None, positions, freqs)
    assert none is None
    check(got, x, positions, freqs, "half")


def test_far_positions_keep_their_angle():
    """Positions near 2^31 and past it: an FP32 angle would be off by whole turns."""
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn(1, 4, 2, 128, generator=g, device=DEV)
    positions = torch.tensor([[2**31 - 1, 2**33 + 5, -(2**31), 0]], device=DEV)
    freqs, _ = tables.rotary_frequencies(128, 10000.0, DEV)
    got, _ = K.rotary(x, None, positions, freqs)
    # the angle itself, a product of 2^33, has an FP64 rounding of 2^-20 radians
    want, tol = rotated(x, positions, freqs, "half")
    assert ((got.double() - want).abs() <= tol + 2.0 ** -19 * x.abs().amax()).all()


@pytest.mark.parametrize("dtype,skew", [(torch.bfloat16, 1), (torch.bfloat16, 4), (torch.float32, 1), (torch.float32, 2)])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_odd_strides_and_alignment(dtype, skew, layout):
    g = torch.Generator(device=DEV).manual_seed(4)
    store = torch.randn(3, 29, 6 * 128 + skew, generator=g, device=DEV).to(dtype)
    x = store[..., skew:].unflatten(-1, (6, 128))
    out = torch.full((3, 29, 6, 128 + skew), 7.0, device=DEV, dtype=dtype)
    view = out[..., skew:].transpose(1, 2)
    freqs, _ = tables.rotary_frequencies(96, 10000.0, DEV)
    positions = torch.arange(29, device=DEV)
    K.rotary(x, None, positions, freqs, layout=layout, q_out=view)
    check(view, x, positions, freqs, layout)
    assert (out[..., :skew] == 7.0).all()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_in_place_and_back(layout, dtype):
    """In place on a packed projection whose other columns stay; and the transposed rotation undoes it."""
    g = torch.Generator(device=DEV).manual_seed(5)
    proj = torch.randn(2, 65, 9 * 128, generator=g, device=DEV).to(dtype)
    before = proj.clone()
    q, k = proj[..., :768].unflatten(-1, (6, 128)), proj[..., 768:1024].unflatten(-1, (2, 128))
    q0, k0 = q.clone(), k.clone()
    freqs, _ = tables.rotary_frequencies(64, 10000.0, DEV)
    positions = torch.arange(65, device=DEV)
    K.rotary(q, k, positions, freqs, layout=layout, q_out=q.transpose(1, 2), k_out=k.transpose(1, 2))
    check(q.transpose(1, 2), q0, positions, freqs, layout)
    check(k.transpose(1, 2), k0, positions, freqs, layout)
    assert torch.equal(proj[..., 1024:], before[..., 1024:])
    back, _ = K.rotary(q, None, positions, freqs, layout=layout, transpose=True)
    tol = 2.1 * (torch.finfo(dtype).eps / 2 + 2.0 ** -21) * (q0.abs().amax() * math.sqrt(2)).item()
    assert ((back.transpose(1, 2).double() - q0.double()).abs() <= tol).all()


def test_gradient_is_the_transposed_rotation():
    """<R x, g> differences against <x, R^T g>, FP32."""
    gen = torch.Generator(device=DEV).manual_seed(6)
    x, d, g = (torch.randn(1, 9, 3, 64, generator=gen, device=DEV) for _ in range(3))
    freqs, factor = tables.rotary_frequencies(48, 10000.0, DEV, "by_parts", 8.0)
    positions = torch.arange(9, device=DEV) + 5000
    for layout in ("half", "interleaved"):
        run = lambda t, **kw: K.rotary(t, None, positions, freqs, layout=layout, factor=factor, **kw)[0]  # noqa: E731
        gx = run(g, transpose=True)
        step = 0.5  # the rotation is linear: any step
        up, down = run(x + step * d), run(x - step * d)
        numeric = ((up - down).double() / (2 * step) * g.transpose(1, 2).double()).sum()
        analytic = (gx.double() * d.transpose(1, 2).double()).sum()
        scale = (d.abs().sum() * g.abs().amax() * factor).double()
        assert (numeric - analytic).abs() <= 2.0 ** -19 * scale


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("token_major", [False, True])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_store_writes_its_rows_only(dtype, token_major, layout):
    g = torch.Generator(device=DEV).manual_seed(7)
    batch, n, heads, kv, dim, rows = 3, 5, 4, 2, 128, 23
    q, k, v = (torch.randn(batch, n, h, dim, generator=g, device=DEV).to(dtype) for h in (heads, kv, kv))
    shape = (batch, rows, kv, dim) if token_major else (batch, kv, rows, dim)
    caches = [torch.randn(shape, generator=g, device=DEV).to(dtype) for _ in range(2)]
    kc, vc = (c.transpose(1, 2) if token_major else c for c in caches)
    k0, v0 = kc.clone(), vc.clone()
    freqs, _ = tables.rotary_frequencies(128, 10000.0, DEV)
    positions = torch.tensor([[0, 1, 2, 3, 4], [100, 101, 102, 103, 104], [7, 8, 9, 10, 11]], device=DEV)
    at = torch.tensor([[0, 1, 2, 3, 4], [22, 20, -1, 23, 5], [-7, 1 << 20, 22, 0, 11]], device=DEV, dtype=torch.int32)
    got = K.rotary_store(q, k, v, positions, freqs, kc, vc, at, layout=layout)
    check(got, q, positions, freqs, layout)
    want_k, tol = rotated(k, positions, freqs, layout)
    for b in range(batch):
        kept = set(range(rows))
        for t in range(n):
            r = at[b, t].item()
            if 0 <= r < rows:
                kept.discard(r)
                assert ((kc[b, :, r].double() - want_k[b, :, t]).abs() <= tol[b, :, t]).all()
                assert torch.equal(vc[b, :, r], v[b, t])
        kept = sorted(kept)
        assert torch.equal(kc[b, :, kept], k0[b, :, kept]) and torch.equal(vc[b, :, kept], v0[b, :, kept])


def test_store_defaults_to_the_positions():
    g = torch.Generator(device=DEV).manual_seed(8)
    q, k, v = (torch.randn(2, 3, h, 64, generator=g, device=DEV).to(torch.bfloat16) for h in (4, 2, 2))
    kc, vc = torch.zeros(2, 2, 16, 64, device=DEV, dtype=torch.bfloat16), torch.zeros(2, 2, 16, 64, device=DEV,
                                                                                       dtype=torch.bfloat16)
    freqs, _ = tables.rotary_frequencies(64, 10000.0, DEV)
    positions = torch.tensor([4, 5, 6], device=DEV)
    K.rotary_store(q, k, v, positions, freqs, kc, vc)
    _, ko = K.rotary(q, k, positions, freqs)
    assert torch.equal(kc[:, :, 4:7], ko) and torch.equal(vc[:, :, 4:7], v.transpose(1, 2))
    assert not kc[:, :, :4].any() and not kc[:, :, 7:].any()


def test_offsets_past_32_bits():
    """Cache rows more than 2^32 bytes apart."""
    rows, stride = 40, 1 << 26
    flat = torch.empty(rows * stride, device=DEV, dtype=torch.bfloat16)
    kc = flat.as_strided((1, 1, rows, 128), (rows * stride, 128, stride, 1))
    vc = flat.as_strided((1, 1, rows, 128), (rows * stride, 128, stride, 1), 256)
    g = torch.Generator(device=DEV).manual_seed(9)
    q, k, v = (torch.randn(1, 2, 1, 128, generator=g, device=DEV).to(torch.bfloat16) for _ in range(3))
    freqs, _ = tables.rotary_frequencies(128, 10000.0, DEV)
    positions = torch.tensor([[3, 39]], device=DEV)
    K.rotary_store(q, k, v, positions, freqs, kc, vc)
    _, ko = K.rotary(q, k, positions, freqs)
    assert torch.equal(kc[:, :, [3, 39]], ko) and torch.equal(vc[:, :, [3, 39]], v.transpose(1, 2))


def test_non_finite_values_stay_in_their_pair():
    g = torch.Generator(device=DEV).manual_seed(10)
    x = torch.randn(1, 3, 2, 128, generator=g, device=DEV).to(torch.bfloat16)
    x[0, 1, 1, 5], x[0, 2, 0, 120] = float("nan"), float("inf")
    freqs, _ = tables.rotary_frequencies(64, 10000.0, DEV)
    y, _ = K.rotary(x, None, torch.arange(3, device=DEV) + 1, freqs)
    bad = ~torch.isfinite(y)
    assert bad.sum() == 3 and bad[0, 1, 1, [5, 37]].all() and y[0, 0, 2, 120] == float("inf")


def test_empty_calls():
    freqs, _ = tables.rotary_frequencies(64, 10000.0, DEV)
    for shape in ((0, 4, 2, 64), (2, 0, 2, 64)):
        x = torch.empty(shape, device=DEV, dtype=torch.bfloat16)
        y, _ = K.rotary(x, None, torch.zeros(shape[1], device=DEV, dtype=torch.int64), freqs)
        assert y.shape == (shape[0], 2, shape[1], 64)


def test_captured_calls_replay():
    """A captured call reads the inputs of each replay, with eager work between."""
    g = torch.Generator(device=DEV).manual_seed(11)
    q, k, v = (torch.randn(2, 1, h, 128, generator=g, device=DEV).to(torch.bfloat16) for h in (4, 2, 2))
    caches = [torch.zeros(2, 2, 16, 128, device=DEV, dtype=torch.bfloat16) for _ in range(4)]
    positions = torch.zeros(2, 1, device=DEV, dtype=torch.int64)
    freqs, _ = tables.rotary_frequencies(128, 10000.0, DEV)
    q_out = torch.empty(2, 4, 1, 128, device=DEV, dtype=torch.bfloat16)
    K.rotary_store(q, k, v, positions, freqs, caches[0], caches[1], q_out=q_out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.rotary_store(q, k, v, positions, freqs, caches[0], caches[1], q_out=q_out)
    caches[0].zero_(), caches[1].zero_()
    for step in range(4):
        for t in (q, k, v):
            t.normal_(generator=g)
        positions.copy_(torch.tensor([[step], [15 - step]]))
        graph.replay()
        want = K.rotary_store(q, k, v, positions, freqs, caches[2], caches[3])
        assert torch.equal(q_out, want)
        assert torch.equal(caches[0], caches[2]) and torch.equal(caches[1], caches[3])


@pytest.mark.parametrize("batch,n,heads", [(1, 3, 2), (2, 1, 3), (2, 3, 1), (1, 1, 1)])
def test_in_place_with_axes_of_one(batch, n, heads):
    """The strides of such axes say nothing: a view that differs from the input only there is the input itself."""
    x = torch.randn(batch, n, heads, 64, generator=torch.Generator(device=DEV).manual_seed(17), device=DEV)
    positions, (freqs, _) = torch.arange(n, device=DEV) + 9, tables.rotary_frequencies(64, 10000.0, DEV)
    before = x.clone()
    strides = [s if size > 1 else 4096 + i for i, (size, s) in enumerate(zip(x.transpose(1, 2).shape, x.transpose(1, 2).stride()))]
    K.rotary(x, None, positions, freqs, q_out=x.transpose(1, 2).as_strided((batch, heads, n, 64), strides))
    check(x.transpose(1, 2), before, positions, freqs, "half")


@pytest.mark.parametrize("batch,n", [(1, 1), (2, 1), (3, 9)])
def test_tensors_that_interleave(batch, n):
    """Query and key heads rotated in place in one projection; K and V caches that alternate row by row and head by head."""
    g = torch.Generator(device=DEV).manual_seed(18)
    proj = torch.randn(batch, n + 2, 8, 64, generator=g, device=DEV).to(torch.bfloat16)[:, 1: n + 1]
    q, k, v = proj[:, :, 0:4], proj[:, :, 4:6], proj[:, :, 6:8]
    positions, (freqs, _) = torch.arange(n, device=DEV) + 5, tables.rotary_frequencies(64, 10000.0, DEV)
    before = proj.clone()
    K.rotary(q, k, positions, freqs, q_out=q.transpose(1, 2), k_out=k.transpose(1, 2))
    check(q.transpose(1, 2), before[:, :, 0:4], positions, freqs, "half")
    check(k.transpose(1, 2), before[:, :, 4:6], positions, freqs, "half")
    assert torch.equal(v, before[:, :, 6:8])
    for shape in ((batch, 20, 2, 2, 64), (batch, 20, 2, 2, 72)):
        caches = torch.zeros(shape, device=DEV, dtype=torch.bfloat16)[..., :64]
        for kc, vc in ((caches[:, :, 0], caches[:, :, 1]), (caches[:, :, :, 0], caches[:, :, :, 1])):
            K.rotary_store(before[:, :, 0:4], before[:, :, 4:6], v, positions, freqs, kc.transpose(1, 2), vc.transpose(1, 2))
            check(kc.transpose(1, 2)[:, :, 5: 5 + n], before[:, :, 4:6], positions, freqs, "half")
            assert torch.equal(vc[:, 5: 5 + n], v) and not kc[:, :5].any() and not vc[:, 5 + n:].any()
            caches.zero_()


def test_an_output_between_its_inputs_rows():
    g = torch.Generator(device=DEV).manual_seed(19)
    packed = torch.randn(2, 7, 4, 64, generator=g, device=DEV)
    before = packed.clone()
    positions, (freqs, _) = torch.arange(7, device=DEV) + 5, tables.rotary_frequencies(64, 10000.0, DEV)
    K.rotary(packed[:, :, 0:2], None, positions, freqs, q_out=packed[:, :, 2:4].transpose(1, 2))
    check(packed[:, :, 2:4].transpose(1, 2), before[:, :, 0:2], positions, freqs, "half")
    assert torch.equal(packed[:, :, 0:2], before[:, :, 0:2])


def test_caches_without_rows():
    g = torch.Generator(device=DEV).manual_seed(20)
    q, k, v = (torch.randn(2, 5, h, 64, generator=g, device=DEV) for h in (4, 2, 2))
    positions, (freqs, _) = torch.arange(5, device=DEV), tables.rotary_frequencies(64, 10000.0, DEV)
    caches = [torch.empty(2, 2, 0, 64, device=DEV) for _ in range(2)]
    check(K.rotary_store(q, k, v, positions, freqs, *caches), q, positions, freqs, "half")
