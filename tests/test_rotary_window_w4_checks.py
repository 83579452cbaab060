"""Refusals of the rotary, windowed attention and 4-bit entry points: wrappers and C ABI, on the CPU."""

import ctypes

import pytest
import torch

from iris_mi355x import _lib
from iris_mi355x import kernels as K
from iris_mi355x import tables

BF16 = torch.bfloat16


@pytest.fixture
def unplaced(monkeypatch):
    """Without the check for GPU tensors, so that the library's own refusals are reached (each comes before
    anything is launched)."""
    monkeypatch.setattr(K, "_on_current_device", lambda op, *tensors: 0)


def test_cpu_tensors_are_refused():
    for call in (attention, rotary, w4):
        with pytest.raises(ValueError, match="GPU"):
            call()


def attention(**change):
    args = dict(q=torch.zeros(2, 4, 3, 128, dtype=BF16), k=torch.zeros(2, 2, 9, 128, dtype=BF16),
                v=torch.zeros(2, 2, 9, 128, dtype=BF16))
    args.update(change)
    return K.window_attention(**args)


@pytest.mark.parametrize("change,match", [
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
def test_window_attention_refuses(unplaced, change, match):
    with pytest.raises(ValueError, match=match):
        attention(**change)


def rotary(**change):
    args = dict(q=torch.zeros(2, 5, 4, 64), k=torch.zeros(2, 5, 2, 64), positions=torch.zeros(2, 5, dtype=torch.int64),
                freqs=torch.zeros(32, dtype=torch.float64))
    args.update(change)
    return K.rotary(**args)


@pytest.mark.parametrize("change,match", [
    (dict(layout="pairs"), "layout"),
    (dict(freqs=torch.zeros(33, dtype=torch.float64)), "33 rotated pairs"),
    (dict(freqs=torch.zeros(0, dtype=torch.float64)), "rotated pairs"),
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
    (dict(k_out=torch.zeros(2, 2, 5, 64, dtype=BF16)), "one dtype"),
    (dict(q_out=torch.zeros(1, 4, 5, 64).expand(2, -1, -1, -1)), "expanded"),
    (dict(q=torch.zeros(2, 5, 4, 64, dtype=torch.float16), k=None), "float32 or bfloat16"),
])
def test_rotary_refuses(unplaced, change, match):
    with pytest.raises(ValueError, match=match):
        rotary(**change)


def test_rotary_refuses_an_output_that_meets_its_input(unplaced):
    x = torch.zeros(2, 6, 4, 64)
    with pytest.raises(ValueError, match="itself"):
        rotary(q=x[:, :5], k=None, q_out=x[:, 1:].transpose(1, 2))
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
def test_gemv_w4_refuses(unplaced, change, match):
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


def test_out_apart_from_inputs(unplaced):
    store = torch.zeros(2, 3, 4, 128, dtype=BF16)
    with pytest.raises(ValueError, match="apart"):
        attention(q=store.transpose(1, 2), out=store.flatten(2))
    x = torch.zeros(128 * 64)
    with pytest.raises(ValueError, match="apart"):
        w4(x=x[:384].view(3, 128), out=x[380:398].view(3, 6))


def test_c_entry_points_refuse():
    """What the library itself turns away, before any launch (pointers are never followed)."""
    at = 1 << 20
    names = {
        "iris_window_attn": (_lib.WINDOW_ATTN_ARGS, dict(
            q=at, k=at, v=at, out=1 << 30, q_shape=(2, 4, 3, 128), q_strides=(1536, 384, 128, 1), k_shape=(2, 2, 9, 128),
            k_strides=(2304, 1152, 128, 1), v_shape=(2, 2, 9, 128), v_strides=(2304, 1152, 128, 1), out_shape=(2, 3, 512),
            out_strides=(1536, 512, 1), window=0, sinks=0, causal=1, lengths=0, lengths_kind=0, starts=0, starts_kind=0,
            start=0, key_mask=0, mask_stride=0, scale=0.1, workspace=0, workspace_bytes=0)),
        "iris_rotary": (_lib.ROTARY_ARGS, dict(
            tensors=1, turned=1, to_rows=3, dtype=0, x=at, x_shape=(2, 5, 2, 64), x_strides=(640, 128, 64, 1), out=1 << 30,
            out_shape=(2, 2, 5, 64), out_strides=(640, 320, 64, 1), rest=(0,) * 36, positions=at, positions_kind=1,
            positions_stride=5, rows=0, rows_kind=0, rows_stride=0, freqs=at, pairs=32, layout=0, transpose=0, factor=1.0)),
        "iris_gemv_w4": (_lib.GEMV_W4_ARGS, dict(
            jobs=1, batch=1, k=128, group=64, x_dtype=0, out_dtype=0, scales_dtype=1, in_act=0, out_act=0, x=at, codes=at,
            scales=at, zeros=0, bias=0, extra_bias=0, out=1 << 30, n=6, n_extra=0, rest=(0,) * 8)),
    }

    def refused(name, match, **change):
        layout, args = names[name]
        values = []
        for value in {**args, **change}.values():
            values += value if isinstance(value, tuple) else (value,)
        with pytest.raises(ValueError, match=match):
            _lib.call(name, layout.pack(*values), None)

    for change, match in ((dict(q_shape=(2, 3, 3, 128)), "multiple"), (dict(k_shape=(2, 2, 1 << 30, 128)), "one shape"),
                          (dict(k_shape=(2, 2, 1 << 30, 128), v_shape=(2, 2, 1 << 30, 128)), "2\\^30"),
                          (dict(window=-1), "negative"), (dict(q=at + 8), "aligned"), (dict(q=0), "null"),
                          (dict(q_strides=(1024, 128, 4, 1)), "strides"), (dict(k_strides=(2304, 1152, 128, 2)), "unit"),
                          (dict(lengths=at, lengths_kind=2), "lengths"), (dict(starts_kind=1), "starts"),
                          (dict(out_strides=(1536, 256, 1)), "overlap"), (dict(out=at), "apart"),
                          (dict(out_shape=(2, 3, 511)), "out must be")):
        refused("iris_window_attn", match, **change)
    for change, match in ((dict(tensors=0), "one to three"), (dict(tensors=4), "one to three"), (dict(dtype=2), "dtype"),
                          (dict(x_shape=(2, 5, 2, 63)), "even"), (dict(pairs=33), "head width"), (dict(layout=2), "layout"),
                          (dict(to_rows=0), "rows"), (dict(positions_kind=2), "positions"),
                          (dict(out_shape=(2, 2, 4, 64)), "output 0"), (dict(x=0), "null"), (dict(freqs=0), "null"),
                          (dict(out=at + 4), "itself"), (dict(out_strides=(0, 320, 64, 1)), "expanded")):
        refused("iris_rotary", match, **change)
    for change, match in ((dict(jobs=3), "one or two"), (dict(group=48), "multiple of 32"), (dict(k=48), "k % 32"),
                          (dict(codes=at + 4), "aligned"), (dict(codes=0), "null"), (dict(n_extra=2), "extra"), (dict(n=0), "rows"),
                          (dict(x=0), "input"), (dict(x=at + 4), "aligned"), (dict(in_act=2), "activation"),
                          (dict(x_dtype=2), "dtype"), (dict(out=at + 8), "apart")):
        refused("iris_gemv_w4", match, **change)
    for name in names:
        with pytest.raises(ValueError, match="null"):
            _lib.call(name, None, None)


def test_rotary_refuses_one_tensor_given_twice(unplaced):
    """The output of one tensor as the input or output of another, which would race."""
    q, k = torch.zeros(2, 5, 2, 64), torch.zeros(2, 5, 2, 64)
    args = (torch.zeros(5, dtype=torch.int64), torch.zeros(32, dtype=torch.float64))
    out = torch.zeros(2, 2, 5, 64)
    with pytest.raises(ValueError, match="another tensor"):
        K.rotary(q, k, *args, q_out=out, k_out=out)
    with pytest.raises(ValueError, match="another tensor"):
        K.rotary(q, k, *args, q_out=k.transpose(1, 2))
    cache = torch.zeros(2, 2, 9, 64)
    with pytest.raises(ValueError, match="another tensor"):
        K.rotary_store(q, k, torch.zeros_like(k), *args, cache, cache)


def test_gemv_w4_pair_refuses_outputs_that_meet(unplaced):
    codes, scales = [torch.zeros(6, 64, dtype=torch.uint8)] * 2, [torch.zeros(6, 2)] * 2
    store = torch.zeros(40)
    with pytest.raises(ValueError, match="lie apart"):
        K.gemv_w4_pair(codes, scales, torch.zeros(3, 128), (None, None), (store[:18].view(3, 6), store[17:35].view(3, 6)))


def test_size_limits():
    """Sizes whose products leave 32 bits, and strides that the kernels' offsets cannot express, are turned away
    before any launch (pointers are never followed)."""
    at, rows = 1 << 20, 1 << 29
    shape = dict(q=at, k=at, v=at, out=1 << 50)

    def attn(name, heads, n_q, n_k, k_stride=128, sinks=0, window=0, batch=1):
        q = (batch, heads, n_q, 128, heads * n_q * 128, n_q * 128, 128, 1)
        k = (batch, 1, n_k, 128, 0, 0, k_stride, 1)
        out = (batch, n_q, heads * 128, n_q * heads * 128, heads * 128, 1)
        args = _lib.WINDOW_ATTN_ARGS.pack(*shape.values(), *q, *k, *k, *out, window, sinks, 1, 0, 0, 0, 0, 0, 0, 0, 0.1, 0, 0)
        if name == "iris_window_attn":
            _lib.call(name, args, None)
            return None
        need = ctypes.c_long(-1)
        _lib.call(name, args, ctypes.byref(need))
        return need.value

    for name in ("iris_window_attn", "iris_window_attn_workspace"):
        with pytest.raises(ValueError, match="2\\^31"):  # (2^32 rows, 0 in 32 bits)
            attn(name, 8, rows, 64)
        with pytest.raises(ValueError, match="not negative"):
            attn(name, 4, 1, 4096, k_stride=-128)
    # the largest sinks count as all keys: the same splits, hence workspace, as without a window
    plain = attn("iris_window_attn_workspace", 4, 1, 65536)
    assert plain > 0 and attn("iris_window_attn_workspace", 4, 1, 65536, sinks=2**63 - 1, window=5) == plain
    with pytest.raises(ValueError, match="workspace"):
        attn("iris_window_attn", 4, 1, 65536)
    with pytest.raises(ValueError, match="too many"):  # a grid of 2^32 threads and more
        attn("iris_window_attn", 16384, 1, 8, batch=16384)
    job = dict(codes=at, scales=at, zeros=0, bias=0, extra_bias=0, out=1 << 50, n=(1 << 30) - 1, n_extra=0)
    with pytest.raises(ValueError, match="too many"):
        _lib.call("iris_gemv_w4", _lib.GEMV_W4_ARGS.pack(2, 1, 32, 32, 0, 0, 1, 0, 0, at, *job.values(),
                                                         *{**job, "out": 1 << 51}.values()), None)
    with pytest.raises(ValueError, match="65536"):
        job.update(n=16, n_extra=65536, extra_bias=at)
        _lib.call("iris_gemv_w4", _lib.GEMV_W4_ARGS.pack(1, 1, 32, 32, 0, 0, 1, 0, 0, at, *job.values(), *(0,) * 8), None)
    tokens = 1 << 28
    head = (at, 1, tokens, 1, 64, 64 * tokens, 64, 64, 1, 1 << 50, 1, 1, tokens, 64, 64 * tokens, 64 * tokens, 64, 1)
    with pytest.raises(ValueError, match="too many"):
        _lib.call("iris_rotary", _lib.ROTARY_ARGS.pack(1, 1, 3, 0, *head, *(0,) * 36, at, 1, 0, 0, 0, 0, at, 32, 0, 0, 1.0), None)


def window_workspace(out_shape, out_strides, heads=4):
    """``iris_window_attn_workspace`` of a call with such an output: its checks of arguments, without a launch."""
    batch, n_q, _ = out_shape
    q = (batch, heads, n_q, 128, heads * n_q * 128, n_q * 128, 128, 1)
    k = (batch, 1, 70, 128, 70 * 128, 70 * 128, 128, 1)
    args = _lib.WINDOW_ATTN_ARGS.pack(1 << 20, 1 << 30, 1 << 31, 1 << 40, *q, *k, *k, *out_shape, *out_strides, 0, 0, 1, 0, 0,
                                      0, 0, 0, 0, 0, 0.1, 0, 0)
    need = ctypes.c_long()
    _lib.call("iris_window_attn_workspace", args, ctypes.byref(need))


@pytest.mark.parametrize("strides", [(512, 512), (1024, 512), (512, 1024), (1024, 1024), (1536, 1024), (516, 1020),
                                     (5120, 516 * 5)])
def test_window_attention_refuses_output_rows_that_overlap(strides):
    """Items that lie fewer rows apart than they have, and rows of two items that meet in part."""
    with pytest.raises(ValueError, match="overlap"):
        window_workspace((3, 5, 512), (*strides, 1))


@pytest.mark.parametrize("strides", [(2560, 512), (512, 1536), (516, 3 * 516), (1024, 4096), (1 << 40, 512), (4096, 680)])
def test_window_attention_takes_output_rows_that_lie_apart(strides):
    """Item or row major, with room between, and rows of items that interleave."""
    window_workspace((3, 5, 512), (*strides, 1))


def test_rotary_refuses_outputs_that_share_memory_in_part(unplaced):
    """An output that meets another tensor's input or output at another address than its first, and one whose own heads do."""
    q, k, v = torch.zeros(2, 5, 2, 64), torch.zeros(2, 5, 2, 64), torch.zeros(2, 5, 2, 64)
    args = (torch.zeros(5, dtype=torch.int64), torch.zeros(32, dtype=torch.float64))
    store = torch.zeros(4096)
    size = 2 * 2 * 5 * 64
    one, two = store[:size].view(2, 2, 5, 64), store[size - 1: 2 * size - 1].view(2, 2, 5, 64)
    for a, b in ((one, two), (two, one)):
        with pytest.raises(ValueError, match="another tensor"):
            K.rotary(q, k, *args, q_out=a, k_out=b)
        with pytest.raises(ValueError, match="another tensor"):
            K.rotary_store(q, k, v, *args, a, b)
        with pytest.raises(ValueError, match="another tensor"):
            K.rotary(q, a.transpose(1, 2), *args, q_out=b)
    packed = torch.zeros(2, 5, 6, 64)  # the heads of a projection, off by one into another tensor's
    with pytest.raises(ValueError, match="another tensor"):
        K.rotary(packed[:, :, 0:2], k, *args, k_out=packed[:, :, 1:3].transpose(1, 2))
    for strides in ((640, 320, 32, 1), (640, 32, 128, 1), (320, 320, 64, 1), (640, 256, 64, 1)):
        with pytest.raises(ValueError, match="overlap"):
            K.rotary(q, None, *args, q_out=store.as_strided((2, 2, 5, 64), strides))


@pytest.mark.parametrize("shape,strides", [((1, 5, 512), (3, 512, 1)), ((3, 1, 512), (516, 7, 1)), ((1, 1, 512), (-1, 2, 1)),
                                           ((3, 1, 512), (1024, 512, 1))])
def test_window_attention_takes_any_output_stride_of_an_axis_of_one(shape, strides):
    window_workspace(shape, strides)


@pytest.mark.parametrize("x,positions,freqs,rows_at", [(0, 1, 1, 1), (1, 0, 1, 1), (1, 1, 0, 1), (1, 1, 1, 0)])
def test_rotary_refuses_null_inputs_of_an_output_without_rows(x, positions, freqs, rows_at):
    """Heads for a cache of no rows are read before their rows are found not to exist."""
    at = 1 << 20
    head = (x * at, 2, 5, 2, 64, 640, 128, 64, 1, 0, 2, 2, 0, 64, 0, 0, 64, 1)
    args = _lib.ROTARY_ARGS.pack(1, 1, 0, 0, *head, *(0,) * 36, positions * at, 1, 5, rows_at * at, 1, 5, freqs * at, 32, 0, 0, 1.0)
    with pytest.raises(ValueError, match="null"):
        _lib.call("iris_rotary", args, None)
