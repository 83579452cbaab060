"""Refusals of the rotary, windowed attention and 4-bit entry points: wrappers and C ABI, on the CPU."""

import pytest
import torch

from iris_mi355x import _lib
from iris_mi355x import kernels as K
from iris_mi355x import tables

BF16 = torch.bfloat16


def attention(**change):
    args = dict(q=torch.zeros(2, 4, 3, 128, dtype=BF16), k=torch.zeros(2, 2, 9, 128, dtype=BF16),
                v=torch.zeros(2, 2, 9, 128, dtype=BF16))
    args.update(change)
    return K.window_attention(**args)


@pytest.mark.parametrize("change,match", [
    (dict(), "GPU"),
    (dict(q=torch.zeros(2, 4, 3, 64, dtype=BF16)), "do not match"),
    (dict(q=torch.zeros(2, 3, 3, 128, dtype=BF16)), "do not match"),
    (dict(q=torch.zeros(1, 4, 3, 128, dtype=BF16)), "do not match"),
    (dict(q=torch.zeros(4, 3, 128, dtype=BF16)), "must be"),
    (dict(q=torch.zeros(2, 4, 3, 128)), "BF16"),
    (dict(v=torch.zeros(2, 2, 8, 128, dtype=BF16)), "one shape"),
    (dict(k=torch.zeros(2, 2, 128, 9, dtype=BF16).transpose(2, 3)), "unit stride"),
    (dict(window=0), "window"),
    (dict(window=-3), "window"),
    (dict(sinks=-1), "sinks"),
    (dict(lengths=torch.zeros(2)), "lengths"),
    (dict(lengths=torch.zeros(3, dtype=torch.int32)), "lengths"),
    (dict(lengths=torch.zeros(4, dtype=torch.int32)[::2]), "lengths"),
    (dict(starts=torch.zeros(2)), "starts"),
    (dict(starts=1 << 61), "starts"),
    (dict(key_mask=torch.zeros(2, 8, dtype=torch.bool)), "key_mask"),
    (dict(key_mask=torch.zeros(2, 9)), "key_mask"),
    (dict(key_mask=torch.zeros(9, 2, dtype=torch.bool).T), "key_mask"),
    (dict(out=torch.zeros(2, 3, 512)), "out"),
    (dict(out=torch.zeros(2, 4, 512, dtype=BF16)), "out"),
])
def test_window_attention_refuses(change, match):
    with pytest.raises(ValueError, match=match):
        attention(**change)


def rotary(**change):
    args = dict(q=torch.zeros(2, 5, 4, 64), k=torch.zeros(2, 5, 2, 64), positions=torch.zeros(2, 5, dtype=torch.int64),
                freqs=torch.zeros(32, dtype=torch.float64))
    args.update(change)
    return K.rotary(**args)


@pytest.mark.parametrize("change,match", [
    (dict(), "GPU"),
    (dict(layout="pairs"), "layout"),
    (dict(freqs=torch.zeros(33, dtype=torch.float64)), "freqs"),
    (dict(freqs=torch.zeros(0, dtype=torch.float64)), "freqs"),
    (dict(freqs=torch.zeros(32)), "freqs"),
    (dict(q=torch.zeros(2, 5, 256)), "heads"),
    (dict(q=torch.zeros(2, 5, 4, 63), k=None, freqs=torch.zeros(4, dtype=torch.float64)), "even"),
    (dict(k=torch.zeros(2, 4, 2, 64)), "heads"),
    (dict(k=torch.zeros(2, 5, 2, 64, dtype=BF16)), "one dtype"),
    (dict(k=torch.zeros(2, 5, 64, 2).transpose(2, 3)), "unit stride"),
    (dict(positions=torch.zeros(2, 5)), "positions"),
    (dict(positions=torch.zeros(5, 2, dtype=torch.int64).T), "positions"),
    (dict(positions=torch.zeros(3, 5, dtype=torch.int64)), "positions"),
    (dict(q_out=torch.zeros(2, 4, 6, 64)), "output 0"),
    (dict(k_out=torch.zeros(2, 2, 5, 64, dtype=BF16)), "output 1"),
    (dict(q_out=torch.zeros(1, 4, 5, 64).expand(2, -1, -1, -1)), "expanded"),
    (dict(q=torch.zeros(2, 5, 4, 64, dtype=torch.float16), k=None), "float32 or bfloat16"),
])
def test_rotary_refuses(change, match):
    with pytest.raises(ValueError, match=match):
        rotary(**change)


def test_rotary_refuses_an_output_that_meets_its_input():
    x = torch.zeros(2, 6, 4, 64)
    with pytest.raises(ValueError, match="itself"):
        rotary(q=x[:, :5], k=None, q_out=x[:, 1:].transpose(1, 2))
    with pytest.raises(ValueError, match="GPU"):  # in place is not refused
        rotary(q=x[:, :5], k=None, q_out=x[:, :5].transpose(1, 2))
    q, k = torch.zeros(2, 5, 4, 64), torch.zeros(2, 5, 2, 64)
    args = (torch.zeros(5, dtype=torch.int64), torch.zeros(32, dtype=torch.float64))
    with pytest.raises(ValueError, match="itself"):  # rows move
        K.rotary_store(q, k, torch.zeros(2, 5, 2, 64), *args, k.transpose(1, 2), torch.zeros(2, 2, 5, 64))
    for rows in (torch.zeros(2, 4, dtype=torch.int64), torch.zeros(2, 5)):
        with pytest.raises(ValueError, match="rows"):
            K.rotary_store(q, k, k, *args, torch.zeros(2, 2, 9, 64), torch.zeros(2, 2, 9, 64), rows)
    with pytest.raises(ValueError, match="output 2"):
        K.rotary_store(q, k, k, *args, torch.zeros(2, 2, 9, 64), torch.zeros(2, 3, 9, 64))


def w4(**change):
    args = dict(codes=torch.zeros(6, 64, dtype=torch.uint8), scales=torch.zeros(6, 2), x=torch.zeros(3, 128),
                bias=torch.zeros(6), out=torch.zeros(3, 6))
    args.update(change)
    return K.gemv_w4(**args)


@pytest.mark.parametrize("change,match", [
    (dict(), "GPU"),
    (dict(codes=torch.zeros(6, 64, dtype=torch.int8)), "codes"),
    (dict(codes=torch.zeros(6, 63, dtype=torch.uint8)), "codes"),
    (dict(codes=torch.zeros(6, 128, dtype=torch.uint8)[:, ::2]), "codes"),
    (dict(group=48), "group"),
    (dict(group=0), "group"),
    (dict(group=128), "scales"),
    (dict(zeros=torch.zeros(6, 2)), "zeros"),
    (dict(zeros=torch.zeros(6, 1, dtype=torch.uint8)), "zeros"),
    (dict(x=torch.zeros(3, 256)[:, ::2]), "contiguous"),
    (dict(x=torch.zeros(128)), "takes"),
    (dict(bias=torch.zeros(5)), "bias"),
    (dict(bias=torch.zeros(6, dtype=BF16)), "bias"),
    (dict(extra_bias=torch.zeros(2, 6)), "out"),
    (dict(extra_bias=torch.zeros(0, 6)), "extra_bias"),
    (dict(out=torch.zeros(6, 3)), "out"),
])
def test_gemv_w4_refuses(change, match):
    with pytest.raises(ValueError, match=match):
        w4(**change)


@pytest.mark.parametrize("lengths", [(1, 2, 2, 2), (2, 1, 2, 2), (2, 2, 3, 2), (2, 2, 2, 0)])
def test_gemv_w4_pair_takes_two_products(lengths):
    codes, scales, biases, outs = ([torch.zeros(1)] * n for n in lengths)
    with pytest.raises(ValueError, match="gemv_w4_pair: takes two products"):
        K.gemv_w4_pair(codes, scales, torch.zeros(1, 64), biases, outs)


@pytest.mark.parametrize("change", [dict(group=48), dict(group=0), dict(weight=torch.zeros(4, 48)), dict(weight=torch.zeros(64))])
def test_pack_w4_refuses(change):
    with pytest.raises(ValueError, match="pack_w4"):
        K.pack_w4(**{"weight": torch.zeros(4, 64), **change})


def test_rotary_frequencies():
    plain, factor = tables.rotary_frequencies(8, 100.0, "cpu")
    assert factor == 1.0 and torch.allclose(plain, torch.tensor([1.0, 100 ** -0.25, 0.1, 100 ** -0.75], dtype=torch.float64))
    linear, factor = tables.rotary_frequencies(8, 100.0, "cpu", "linear", 4.0)
    assert factor == 1.0 and torch.equal(linear, plain / 4)
    ntk, factor = tables.rotary_frequencies(8, 100.0, "cpu", "ntk", 4.0)
    assert factor == 1.0 and ntk[0] == 1.0 and torch.allclose(ntk[-1], plain[-1] / 4)
    parts, factor = tables.rotary_frequencies(128, 10000.0, "cpu", "by_parts", 8.0, trained=4096)
    plain, _ = tables.rotary_frequencies(128, 10000.0, "cpu")
    turns = 4096 * plain / (2 * torch.pi)
    assert torch.equal(parts[turns >= 32], plain[turns >= 32])
    assert torch.allclose(parts[turns <= 1], plain[turns <= 1] / 8, rtol=1e-15, atol=0)
    between = (turns > 1) & (turns < 32)
    assert between.any() and (parts[between] < plain[between]).all() and (parts[between] > plain[between] / 8).all()
    assert abs(factor - 1.2079441541679836) < 1e-15
    for bad in (dict(dim=7), dict(dim=0), dict(scaling="cubic"), dict(scale=0.5), dict(scale=2.0), dict(theta=1.0),
                dict(scaling="by_parts", slow=4.0, fast=4.0)):
        with pytest.raises(ValueError, match="rotary_frequencies"):
            tables.rotary_frequencies(**{"dim": 8, "theta": 100.0, "device": "cpu", **bad})


def test_c_entry_points_refuse():
    """What the library itself turns away, before any launch (pointers are never followed)."""
    at = 1 << 20
    longs, ints, pointers = _lib.long_array, _lib.int_array, _lib.pointer_array
    s3 = longs([1024, 128, 128])

    def attn(q=at, heads=4, kv=2, nq=3, nk=9, window=0, sinks=0, qs=s3, lengths_kind=0, lengths=None, starts=None,
             starts_kind=0):
        _lib.call("iris_window_attn", q, qs, at, s3, at, s3, at, longs([2048, 512]), 2, heads, kv, nq, nk, window, sinks, 1,
                  lengths, lengths_kind, starts, starts_kind, 0, None, 0, 0.1, None)

    for change, match in ((dict(heads=3), "multiple"), (dict(nk=1 << 30), "2\\^30"), (dict(window=-1), "negative"),
                          (dict(q=at + 8), "aligned"), (dict(q=None), "null"), (dict(qs=longs([1024, 128, 4])), "strides"),
                          (dict(lengths=at, lengths_kind=2), "lengths"), (dict(starts_kind=1), "starts")):
        with pytest.raises(ValueError, match=match):
            attn(**change)

    def turn(tensors=1, dim=64, pairs=32, layout=0, flags=1, rows=None, kind=1, out_rows=5, x=at):
        _lib.call("iris_rotary", tensors, pointers([x]), longs([640, 128, 64]), pointers([at]), longs([640, 320, 64]),
                  ints([2]), ints([flags]), longs([out_rows]), _lib.F32, 2, 5, dim, at, kind, 5, rows, 1, 0, at, pairs,
                  layout, 1.0, 0, None)

    for change, match in ((dict(tensors=0), "one to three"), (dict(tensors=4), "one to three"), (dict(dim=63), "even"),
                          (dict(pairs=33), "head width"), (dict(layout=2), "layout"), (dict(flags=3), "rows"),
                          (dict(kind=2), "positions"), (dict(out_rows=4), "fewer rows"), (dict(x=None), "null")):
        with pytest.raises(ValueError, match=match):
            turn(**change)

    def gemv(jobs=1, group=64, k=128, codes=at, extra=0, x=at, act=0):
        _lib.call("iris_gemv_w4", jobs, pointers([codes]), pointers([at]), _lib.BF16, pointers([None]), group, x, _lib.F32,
                  1, ints([6]), k, pointers([None]), pointers([None]), ints([extra]), pointers([at]), _lib.F32, act, 0, None)

    for change, match in ((dict(jobs=3), "one or two"), (dict(group=48), "multiple of 32"), (dict(k=48), "k % 32"),
                          (dict(codes=at + 4), "aligned"), (dict(codes=None), "null"), (dict(extra=2), "extra"),
                          (dict(x=None), "input"), (dict(act=2), "activation")):
        with pytest.raises(ValueError, match=match):
            gemv(**change)
