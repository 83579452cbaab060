"""``gemv_w4`` / ``gemv_w4_pair`` against FP64: group sizes, zero points, ragged last groups, row and batch
edges, types, activations, extra biases."""

import pytest
import torch

from iris_mi355x import kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(seed, n, k, group, batch, zeros, scales_dtype=torch.bfloat16, x_dtype=torch.float32, extra=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    groups = -(-k // group)
    codes = torch.randint(0, 256, (n, k // 2), generator=g, device=DEV, dtype=torch.uint8)
    scales = (0.02 * torch.randn(n, groups, generator=g, device=DEV)).to(scales_dtype)
    z = torch.randint(0, 16, (n, groups), generator=g, device=DEV, dtype=torch.uint8) if zeros else None
    x = torch.randn(batch, k, generator=g, device=DEV).to(x_dtype)
    bias = torch.randn(n, generator=g, device=DEV)
    add = torch.randn(extra, n, generator=g, device=DEV) if extra else None
    return codes, scales, z, x, bias, add


def weights(codes, scales, z, group):
    w = torch.stack([codes & 15, codes >> 4], -1).flatten(1).double()
    of = torch.arange(w.shape[1], device=DEV) // group
    return (w - (8.0 if z is None else z.double()[:, of])) * scales.double()[:, of]


def expected(codes, scales, z, x, bias, add, group, in_silu=False, out_silu=False, out_dtype=torch.float32):
    """``(y, tolerance)`` in FP64. FP32 sums of a group's products with codes offset by up to 16 + 15, then of
    the groups and of a few partial sums: the depth times 2^-24 of the absolute sum at worst (the inputs
    themselves are exact, or carry silu's few 2^-23); half a step of the output type."""
    w = weights(codes, scales, z, group)
    xd = x.double()
    xd = torch.nn.functional.silu(xd) if in_silu else xd
    y = xd @ w.T
    of = torch.arange(w.shape[1], device=DEV) // group
    spread = xd.abs() @ (62.0 * scales.double().abs()[:, of]).T
    tol = (group + scales.shape[1] + 24) * 2.0 ** -24 * spread
    if in_silu:
        tol = tol + 2.0 ** -20 * (xd.abs() @ w.abs().T)
    if bias is not None:
        y = y + bias.double()
    if out_silu:
        y = torch.nn.functional.silu(y)
        tol = 1.2 * tol + 2.0 ** -20 * y.abs()
    if add is not None:
        y = y + add.double()[:, None]
    return y, tol + (torch.finfo(out_dtype).eps / 2 + 2.0 ** -23) * y.abs()


def check(out, args, group, **options):
    codes, scales, z, x, bias, add = args
    want, tol = expected(codes, scales, z, x, bias, add, group, out_dtype=out.dtype, **options)
    err = (out.double() - want).abs()
    assert (err <= tol).all(), f"worst {(err / tol).max().item():.3g} of the tolerance"
    if out.dtype == torch.float32:  # and in norm: roundings that fall either way
        assert err.norm() <= 4e-6 * (want.norm() + 1e-30)


def run(args, group, out_dtype=None, **options):
    codes, scales, z, x, bias, add = args
    shape = (x.shape[0], codes.shape[0])
    out = torch.full((add.shape[0], *shape) if add is not None else shape, 7.0, device=DEV, dtype=out_dtype or x.dtype)
    assert K.gemv_w4(codes, scales, x, bias, out, group=group, zeros=z, extra_bias=add, **options) is out
    return out


@pytest.mark.parametrize("n", [1, 15, 16, 17, 63, 65, 200, 1000])
@pytest.mark.parametrize("k,group", [(32, 32), (64, 64), (96, 64), (128, 32), (160, 128), (256, 256), (544, 32), (2560, 64),
                                     (2592, 128), (6848, 128)])
@pytest.mark.parametrize("zeros", [False, True])
def test_sizes(n, k, group, zeros):
    args = make(40, n, k, group, 1, zeros)
    check(run(args, group), args, group)


@pytest.mark.parametrize("batch", [1, 2, 3, 4, 5, 6, 8, 11, 16, 17, 21, 22, 32, 33, 64, 65, 130])
@pytest.mark.parametrize("x_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,k,group", [(40, 192, 64), (130, 1312, 32), (33, 640, 128)])
def test_batches(batch, x_dtype, n, k, group):
    args = make(41, n, k, group, batch, True, x_dtype=x_dtype)
    check(run(args, group), args, group)


@pytest.mark.parametrize("x_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scales_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("batch", [1, 7])
def test_types_activations_and_extra_biases(x_dtype, out_dtype, scales_dtype, batch):
    for extra in (0, 1, 9):
        for bias in (True, False):
            args = make(42, 150, 704, 64, batch, extra == 9, scales_dtype, x_dtype, extra)
            if not bias:
                args = (*args[:4], None, args[5])
            for acts in ({}, {"in_silu": True}, {"out_silu": True}, {"in_silu": True, "out_silu": True}):
                check(run(args, 64, out_dtype, **acts), args, 64, **acts)


@pytest.mark.parametrize("n", [2560, 15360])
@pytest.mark.parametrize("batch", [1, 2, 24])
def test_wide(n, batch):
    args = make(43, n, 2560, 64, batch, False, extra=3)
    check(run(args, 64, in_silu=True), args, 64, in_silu=True)


@pytest.mark.parametrize("ns", [(15360, 15360), (40, 24), (1, 300)])
@pytest.mark.parametrize("batch", [1, 2, 9, 70])
def test_pair_is_two_calls(ns, batch):
    jobs = [make(44 + i, n, 320, 64, batch, i == 1, extra=j) for i, (n, j) in enumerate(zip(ns, (5, 2)))]
    x = jobs[0][3]
    outs = [[torch.full((a[5].shape[0], batch, a[0].shape[0]), 7.0, device=DEV) for a in jobs] for _ in range(2)]
    K.gemv_w4_pair([a[0] for a in jobs], [a[1] for a in jobs], x, [a[4] for a in jobs], outs[0], 64,
                   [a[2] for a in jobs], [a[5] for a in jobs], in_silu=True)
    for a, out in zip(jobs, outs[1]):
        K.gemv_w4(a[0], a[1], x, a[4], out, 64, a[2], a[5], in_silu=True)
    for got, want, a in zip(*outs, jobs):
        assert torch.equal(got, want)
        check(got, (*a[:3], x, *a[4:]), 64, in_silu=True)


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_non_finite_values_stay_in_their_row(value):
    """An infinite scale reaches its weight row, a NaN input its batch row, and nothing else."""
    codes, scales, z, x, bias, _ = make(46, 50, 256, 32, 7, False)
    out = run((codes, scales, z, x, bias, None), 32)
    codes[7, 0] = 0x11  # not the zero point
    scales[7, 0] = value
    got = run((codes, scales, z, x, bias, None), 32)
    assert not torch.isfinite(got[:, 7]).any() and torch.equal(got[:, :7], out[:, :7]) and torch.equal(got[:, 8:], out[:, 8:])
    scales[7, 0] = 0.01
    x[4, 100] = value
    got = run((codes, scales, z, x, bias, None), 32)
    assert not torch.isfinite(got[4][[i for i in range(50) if codes[i, 50] & 15 != 8]]).any()
    others = [0, 1, 2, 3, 5, 6]
    assert torch.isfinite(got[others]).all()


def test_large_and_small_inputs():
    """FP32 inputs over the whole exponent range that their products allow."""
    codes, scales, z, x, bias, _ = make(47, 64, 512, 64, 3, True)
    x[0] *= 1e30
    x[1] *= 1e-30
    args = (codes, scales, z, x, None, None)
    out = run(args, 64)
    want, tol = expected(codes, scales, z, x, None, None, 64)
    assert ((out.double() - want).abs() <= tol).all()
    for b in range(3):
        assert (out[b].double() - want[b]).norm() <= 4e-6 * want[b].norm()


@pytest.mark.parametrize("symmetric", [True, False])
def test_packed_weights(symmetric):
    """``pack_w4``: every weight within half a step of its code, and the product of the packed weights."""
    g = torch.Generator(device=DEV).manual_seed(48)
    w = torch.randn(70, 288, generator=g, device=DEV)
    w[3] = 0.0
    w[4, :64] = w[4, :64].abs() + 1  # a group of one sign
    codes, scales, zeros = K.pack_w4(w, 64, symmetric)
    back = weights(codes, scales, zeros, 64)
    of = torch.arange(288, device=DEV) // 64
    step = scales.double()[:, of]
    # half a step, and what the scale's rounding to BF16 (2^-8) and, with a zero point, its rounding clip at the ends
    slack = 8 * 2.0 ** -8 if symmetric else 0.5 + 16 * 2.0 ** -8
    assert ((back - w.double()).abs() <= (0.5 + slack) * step + 1e-7).all()
    x = torch.randn(2, 288, generator=g, device=DEV)
    args = (codes, scales, zeros, x, None, None)
    check(run(args, 64), args, 64)


def test_captured_calls_replay():
    args = make(49, 300, 640, 64, 2, True, extra=2)
    codes, scales, z, x, bias, add = args
    out = torch.empty(2, 2, 300, device=DEV)
    K.gemv_w4(codes, scales, x, bias, out, 64, z, add)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.gemv_w4(codes, scales, x, bias, out, 64, z, add)
    g = torch.Generator(device=DEV).manual_seed(50)
    for _ in range(3):
        x.normal_(generator=g)
        out.zero_()
        graph.replay()
        assert torch.equal(out, run(args, 64))


def test_empty_batch():
    codes, scales, z, x, bias, _ = make(51, 20, 64, 64, 1, False)
    out = torch.empty(0, 20, device=DEV)
    K.gemv_w4(codes, scales, x[:0], bias, out)


@pytest.mark.parametrize("extra,batch", [(65535, 2), (9000, 32), (1, 33)])
def test_many_extra_biases(extra, batch):
    args = make(49, 17, 64, 32, batch, True, x_dtype=torch.bfloat16, extra=extra)
    check(run(args, 32, torch.float32), args, 32)


@pytest.mark.parametrize("batch,k,x_dtype,in_silu", [
    (1, 81920, torch.bfloat16, False), (16, 9984, torch.bfloat16, False), (27, 6848, torch.bfloat16, False),
    (32, 12288, torch.bfloat16, False), (1, 30016, torch.float32, False), (5, 8192, torch.float32, True),
    (9, 6880, torch.float32, False), (16, 4128, torch.float32, True), (5, 9984, torch.bfloat16, True),
    (16, 9984, torch.bfloat16, True)])
@pytest.mark.parametrize("group", [32, 128, 4096])
@pytest.mark.parametrize("n", [40, 2100])
def test_k_in_stages(batch, k, x_dtype, in_silu, group, n):
    """Inputs that fill more than a workgroup's LDS, few and many waves side by side."""
    args = make(50, n, k, group, batch, True, x_dtype=x_dtype)
    check(run(args, group, torch.float32, in_silu=in_silu), args, group, in_silu=in_silu)


@pytest.mark.parametrize("batch,k,x_dtype", [(16, 9984, torch.bfloat16), (28, 4992, torch.bfloat16), (4, 8192, torch.float32),
                                             (14, 2592, torch.float32)])
def test_k_in_stages_of_many_rows(batch, k, x_dtype):
    args = make(51, 30001, k, 64, batch, False, x_dtype=x_dtype)
    check(run(args, 64, torch.float32), args, 64)


def test_pair_of_which_one_takes_stages():
    jobs = [make(52 + i, n, 4096, 64, 4, False) for i, n in enumerate((30000, 40))]
    x = jobs[0][3]
    outs = [[torch.full((4, a[0].shape[0]), 7.0, device=DEV) for a in jobs] for _ in range(2)]
    K.gemv_w4_pair([a[0] for a in jobs], [a[1] for a in jobs], x, [a[4] for a in jobs], outs[0], 64)
    for a, out, got in zip(jobs, outs[1], outs[0]):
        K.gemv_w4(a[0], a[1], x, a[4], out, 64)
        assert torch.equal(got, out)
        check(got, (*a[:3], x, *a[4:]), 64)


@pytest.mark.parametrize("batch,x_dtype,ns", [
    (4, torch.float32, (30000, 40)), (5, torch.float32, (30000, 40)), (5, torch.float32, (40, 30000)),
    (8, torch.bfloat16, (28672, 1024)), (9, torch.bfloat16, (28672, 1024)), (16, torch.bfloat16, (28672, 1024)),
    (16, torch.bfloat16, (1024, 28672)), (16, torch.bfloat16, (15360, 1280))])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_pair_in_stages_is_two_calls(batch, x_dtype, ns, group):
    """One product of a pair in stages of k, the other whole: with more inputs than a stage's first registers hold."""
    jobs = [make(54 + i, n, 4096, group, batch, i == 1, x_dtype=x_dtype) for i, n in enumerate(ns)]
    x = jobs[0][3]
    outs = [[torch.full((batch, a[0].shape[0]), 7.0, device=DEV) for a in jobs] for _ in range(2)]
    K.gemv_w4_pair([a[0] for a in jobs], [a[1] for a in jobs], x, [a[4] for a in jobs], outs[0], group,
                   [a[2] for a in jobs])
    for a, out, got in zip(jobs, outs[1], outs[0]):
        K.gemv_w4(a[0], a[1], x, a[4], out, group, a[2])
        assert torch.equal(got, out)
        check(got, (*a[:3], x, *a[4:]), group)


def product_by_product(args, group, in_silu=False):
    """The formula in FP64 with every infinity and NaN where it puts them."""
    codes, scales, z, x, bias, _ = args
    xd = torch.nn.functional.silu(x.double()) if in_silu else x.double()
    return (xd[:, None, :] * weights(codes, scales, z, group)).sum(-1) + bias.double()


@pytest.mark.parametrize("x_dtype,batch", [(torch.float32, 20), (torch.bfloat16, 40), (torch.bfloat16, 7)])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("in_silu", [False, True])
def test_non_finite_values_give_what_the_formula_has(x_dtype, batch, zeros, in_silu):
    """Infinities of either sign by the signs of weights and inputs, NaN only where an infinity meets its opposite, a zero or
    a NaN; in later pieces of the rows, in a short last group."""
    args = make(55, 70, 288, 128, batch, zeros, x_dtype=x_dtype)
    codes, scales, z, x, bias, _ = args
    inf, nan = float("inf"), float("nan")
    x[batch - 1, 100], x[batch - 2, 287] = inf, -inf
    x[0, 3], x[0, 200] = inf, -inf
    x[2, 7], x[batch - 4, 0] = nan, -inf
    scales[7, 2], scales[9, 0], scales[11, 1] = inf, -inf, nan
    want = product_by_product(args, 128, in_silu)
    got = run(args, 128, torch.float32, in_silu=in_silu).double()
    assert (want == inf).any() and (want == -inf).any() and want.isnan().any() and want.isfinite().any()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got[want.isinf()], want[want.isinf()])
    _, tol = expected(*args, 128, in_silu=in_silu)
    assert ((got - want).abs() <= tol)[want.isfinite()].all()


@pytest.mark.parametrize("x_dtype,batch", [(torch.float32, 17), (torch.bfloat16, 33), (torch.bfloat16, 1)])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("in_silu", [False, True])
def test_finite_results_of_offset_products_that_overflow(x_dtype, batch, zeros, in_silu):
    """Inputs around 1e37 of one sign with small scales: 32 of them times 16 leave FP32, the result does not.

    Such results are FP32 sums, lane by lane, of k / 64 products and over 64 lanes, the weight and each product rounded once:
    (k / 64 + 6 + 2) 2^-24 of their absolute sum, a few 2^-23 for silu."""
    codes, scales, z, x, bias, _ = make(56, 70, 288, 128, batch, zeros, x_dtype=x_dtype)
    x = ((1 + x.float().abs()) * 1e37).to(x_dtype)
    scales = (0.01 * scales.float()).to(scales.dtype)
    args = (codes, scales, z, x, bias, None)
    assert 16 * x.double()[:, :32].sum(1).min() > torch.finfo(torch.float32).max
    w = weights(codes, scales, z, 128)
    want = x.double() @ w.T + bias.double()
    tol = (13 + (16 if in_silu else 0)) * 2.0 ** -24 * (x.double() @ w.abs().T) + 2.0 ** -23 * want.abs()
    assert want.abs().max() < torch.finfo(torch.float32).max
    got = run(args, 128, torch.float32, in_silu=in_silu).double()
    assert ((got - want).abs() <= tol).all()


@pytest.mark.parametrize("batch", [1, 2, 9, 33])
@pytest.mark.parametrize("zeros", [False, True])
def test_codes_at_the_zero_point_under_large_inputs(batch, zeros):
    """Most weights zero, inputs of one sign with a few far above the others: the sums of x (16 + code) and x (16 + zero),
    which the bound of ``expected`` counts whatever their difference, cancel almost whole."""
    codes, scales, z, x, bias, _ = make(57, 150, 1312, 32, batch, zeros)
    g = torch.Generator(device=DEV).manual_seed(58)
    of = torch.arange(1312, device=DEV) // 32
    zero = z[:, of] if zeros else torch.full((150, 1312), 8, device=DEV, dtype=torch.uint8)
    code = torch.stack([codes & 15, codes >> 4], -1).flatten(1)
    code = torch.where(torch.rand(150, 1312, generator=g, device=DEV) < 0.9, zero, code)
    codes = (code[:, 0::2] | code[:, 1::2] << 4).contiguous()
    x = x.abs()
    x[:, [3, 700, 1311]] *= torch.tensor([1e3, 1e4, 3e3], device=DEV)
    args = (codes, scales, z, x, bias, None)
    want, tol = expected(*args, 32)
    got = run(args, 32).double()
    assert ((got - want).abs() <= tol).all()
    code[:, [3, 700, 1311]] = zero[:, [3, 700, 1311]]  # the large inputs meet zeros alone
    codes = (code[:, 0::2] | code[:, 1::2] << 4).contiguous()
    args = (codes, scales, z, x, bias, None)
    want, tol = expected(*args, 32)
    got = run(args, 32).double()
    assert ((got - want).abs() <= tol).all()
