"""The operators for training and serving beside the path: the scaled lookup, the table's gradient, the gradient of the
RMS norm, and the head norms with rotation with their gradient.

Each is compared with its formula in 64 bits on the same inputs.  Tolerances: a result of type T is off by half a step
of T (``finfo(T).eps / 2`` of its size, and half the smallest subnormal) plus the error of the f32 arithmetic before
that rounding.  With u = 2^-24, an f32 sum of terms t_i in any order with at most D additions on a path is off by at most
D u sum|t_i|, and every further operation adds u of its result.  The bounds below count those: SUM(n) is the longest path
of an n-term row sum (n / 32 terms per lane, then 5 + 5 steps over lanes and warps), OPS the products, the square root
and the divisions around it.  Sums of small whole numbers are exact in f32 and are compared for equality."""
import math

import numpy as np
import pytest
import torch

U = 2.0 ** -24
OPS = 16
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def SUM(n):
    return n / 32 + 10


def rounding(dtype):
    """(relative, absolute) half step of a type."""
    f = torch.finfo(dtype)
    return f.eps / 2, f.smallest_normal * f.eps / 2


def check(got, want, inner):
    """got (type T) against want (64 bits), `inner` bounding the f32 error before the rounding to T."""
    rel, least = rounding(got.dtype)
    got = got.double()
    bound = inner + rel * (want.abs() + inner) + least
    bad = ~((got - want).abs() <= bound)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {((got - want).abs() / bound).max().item():.3g} of the bound"


def rand(seed, shape, dtype, mean=0.0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g, dtype=torch.float64) * std + mean).to(dtype).cuda()


def make_ids(seed, n, vocab, kind, id_dtype=torch.int64):
    g = torch.Generator().manual_seed(seed)
    if kind == "same":
        ids = torch.full((n,), vocab // 2)
    elif kind == "skew":
        ids = (vocab * torch.rand(n, generator=g, dtype=torch.float64) ** 6).long()
    elif kind == "falling":
        ids = (vocab - 1 - torch.arange(n)) % vocab
    else:
        ids = torch.randint(0, vocab, (n,), generator=g)
    if id_dtype == torch.uint32:
        return ids.to(torch.int32).view(torch.uint32).cuda()
    return ids.to(id_dtype).cuda()


def as_long(ids):
    return (ids.view(torch.int32) if ids.dtype == torch.uint32 else ids).long()


# ---- refusals, decided on the host -------------------------------------------------------------------------


def test_refusals_need_no_device():
    import candle_b200 as cb

    table, ids = torch.zeros(10, 8), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(cb.CandleError, match="no CPU fallback"):
        cb.embedding_scaled(table, ids, 2.0)
    with pytest.raises(cb.CandleError, match="contiguous"):
        cb.embedding_scaled(table.t(), ids, 2.0)
    with pytest.raises(cb.CandleError, match="unsupported dtype"):
        cb.embedding_scaled(table.double(), ids, 2.0)
    with pytest.raises(cb.CandleError, match="ids"):
        cb.embedding_scaled(table, ids.float(), 2.0)

    grad = torch.zeros(3, 8)
    with pytest.raises(cb.CandleError, match="no CPU fallback"):
        cb.embedding_backward(grad, ids, 10)
    with pytest.raises(cb.CandleError, match="shape mismatch"):
        cb.embedding_backward(torch.zeros(4, 8), ids, 10)
    with pytest.raises(cb.CandleError, match="one stride"):
        cb.embedding_backward(torch.zeros(3, 2, 8).transpose(0, 1), torch.zeros(2, 3, dtype=torch.int64), 10)
    with pytest.raises(cb.CandleError, match="last dimension"):
        cb.embedding_backward(torch.zeros(8, 3).t(), ids, 10)
    with pytest.raises(cb.CandleError, match="unsupported dtype"):
        cb.embedding_backward(grad, ids, 10, out_dtype=torch.bfloat16)
    with pytest.raises(cb.CandleError, match="-1 rows"):
        cb.embedding_backward(grad, ids, -1)

    x, w = torch.zeros(4, 8), torch.ones(8)
    with pytest.raises(cb.CandleError, match="no CPU fallback"):
        cb.rms_norm_backward(x, x, w, 1e-5)
    with pytest.raises(cb.CandleError, match="shape mismatch in rms-norm-backward"):
        cb.rms_norm_backward(torch.zeros(3, 8), x, w, 1e-5)
    with pytest.raises(cb.CandleError, match="shape mismatch in rms-norm-backward"):
        cb.rms_norm_backward(x.half(), x, w, 1e-5)
    with pytest.raises(cb.CandleError, match="has to be contiguous"):
        cb.rms_norm_backward(torch.zeros(8, 4).t(), x, w, 1e-5)
    with pytest.raises(cb.CandleError, match="shape mismatch in rms-norm "):
        cb.rms_norm_backward(x, x, torch.ones(7), 1e-5)

    q, k, wd, cs = torch.zeros(5, 4, 16), torch.zeros(5, 2, 16), torch.ones(16), torch.ones(5, 8)
    with pytest.raises(cb.CandleError, match="no CPU fallback"):
        cb.qk_norm_rope(q, k, wd, wd, 1e-5, cs, cs)
    for bad in (
        dict(k=torch.zeros(4, 2, 16)), dict(k=torch.zeros(5, 2, 8)), dict(k=torch.zeros(1, 5, 2, 16)),
        dict(k=k.half()), dict(q_weight=torch.ones(15)), dict(q_weight=wd.half()), dict(cos=torch.ones(4, 8), sin=torch.ones(4, 8)),
        dict(cos=torch.ones(5, 9), sin=torch.ones(5, 9)), dict(sin=torch.ones(5, 7)), dict(cos=cs.half(), sin=cs.half()),
        dict(q=torch.zeros(5, 16, 4).transpose(1, 2)), dict(positions=torch.zeros(4, dtype=torch.int64)),
        dict(positions=torch.zeros(5)), dict(positions=torch.zeros(10, dtype=torch.int64)[::2]),
        dict(out=(q, torch.zeros(5, 3, 16))), dict(cos=torch.ones(8, 5).t()),
    ):
        a = dict(q=q, k=k, q_weight=wd, k_weight=wd, cos=cs, sin=cs, positions=None, out=None) | bad
        with pytest.raises(cb.CandleError, match="(?!.*no CPU fallback)"):
            cb.qk_norm_rope(a["q"], a["k"], a["q_weight"], a["k_weight"], 1e-5, a["cos"], a["sin"], positions=a["positions"], out=a["out"])
    with pytest.raises(cb.CandleError, match="shape mismatch in qk-norm-rope-backward"):
        cb.qk_norm_rope_backward(q[:4], k, q, k, wd, wd, 1e-5, cs, cs)


def test_overlapping_outputs_are_told_apart():
    from candle_b200 import CandleError
    from candle_b200.ops import _check_apart

    qkv = torch.zeros(2, 7, 10, 16)  # 6 + 2 + 2 heads, packed
    q, k, v = qkv[:, :, :6], qkv[:, :, 6:8], qkv[:, :, 8:]
    for a, b in ((q, k), (k, q), (v, q), (q, v), (k, v)):
        _check_apart("x", a, b, same=False)
    head_major = torch.zeros(2, 10, 7, 16)
    _check_apart("x", head_major[:, :6].transpose(1, 2), head_major[:, 6:8].transpose(1, 2), same=False)
    _check_apart("x", q, q)
    for a, b in ((q, qkv[:, :, 5:8]), (q, qkv[:, :, 1:7]), (qkv[:, 1:], qkv[:, :-1]), (q[:, :, :, :8], q[:, :, :, 4:12])):
        with pytest.raises(CandleError, match="overlaps"):
            _check_apart("x", a, b)
    with pytest.raises(CandleError, match="overlaps"):
        _check_apart("x", q, q, same=False)
    flat = torch.zeros(100)
    _check_apart("x", flat[:50], flat[50:])
    with pytest.raises(CandleError, match="overlaps"):
        _check_apart("x", flat[:51], flat[50:])


def test_overlapping_views_with_broadcast_dimensions_are_refused():
    from candle_b200 import CandleError
    from candle_b200.ops import _check_apart

    b = torch.zeros(12)
    rows = torch.zeros(3, 8)
    for x, y in ((b[:8].expand(4, 8), b[4:12].expand(4, 8)), (b[:8].expand(1, 8), b[4:12].expand(4, 8)),
                 (b[:8].expand(2, 4, 8), b[7:].expand(2, 4, 5)), (rows[:2, None].expand(2, 4, 8), rows[1:, None].expand(2, 4, 8))):
        with pytest.raises(CandleError, match="overlaps"):
            _check_apart("x", x, y)
    # columns of the same rows, each read for all heads
    _check_apart("x", rows[:, None, :4].expand(3, 4, 4), rows[:, None, 4:].expand(3, 4, 4), same=False)


def test_the_same_view_whatever_the_strides_of_its_single_dimensions():
    from candle_b200 import CandleError
    from candle_b200.ops import _check_apart

    one = torch.zeros(6, 4, 16)  # a decoding step's heads: one token each, in two orders of the same memory
    q, seen = one.unsqueeze(1), one.unsqueeze(2).transpose(1, 2)
    assert q.shape == seen.shape and q.stride() != seen.stride()
    _check_apart("x", q, seen)
    _check_apart("x", seen[:1], q[:1])
    row = torch.zeros(5, 64)
    _check_apart("x", row[2:3], row[2:3].as_strided((1, 64), (7, 1), row[2:3].storage_offset()))
    for other in (q[:, :, :3], q[1:], seen.transpose(1, 2), q.view(torch.int32)):
        with pytest.raises(CandleError, match="overlaps"):
            _check_apart("x", q, other)
    with pytest.raises(CandleError, match="overlaps"):
        _check_apart("x", q, seen, same=False)


def test_c_entry_points_refuse_on_the_host():
    import ctypes
    import struct

    from candle_b200 import _cabi
    from candle_b200.ops import _HEADS, _QK_ARGS

    lib, one = _cabi.lib, ctypes.c_void_p(16)  # never dereferenced: validation fails first
    n = ctypes.c_int64()
    assert lib.cb200_embedding_scaled(one, one, one, 10, 8, 2, 1.0, 7, 1, None, None) == -2
    assert lib.cb200_embedding_scaled(one, one, one, 10, 8, 2, 1.0, 0, 9, None, None) == -2
    assert lib.cb200_embedding_scaled(None, one, one, 10, 8, 2, 1.0, 0, 1, None, None) == -1
    assert lib.cb200_embedding_backward_workspace(10, 8, 1 << 31, ctypes.addressof(n)) == -5
    assert lib.cb200_embedding_backward_workspace(10, 8, 100, ctypes.addressof(n)) == 0 and n.value > 1600
    args = [one, 8, one, one, 10, 8, 100, 1.0, -1, 0, 0, 0, 1, one, n.value, None, None]
    for i, bad in ((0, None), (1, -1), (3, None), (4, -1), (10, 5), (11, 2), (12, 7), (13, None), (13, ctypes.c_void_p(8)), (14, n.value - 1)):
        assert lib.cb200_embedding_backward(*(bad if j == i else a for j, a in enumerate(args))) < 0, i
    assert lib.cb200_rms_norm_backward_workspace(4, 0, ctypes.addressof(n)) == -1
    assert lib.cb200_rms_norm_backward_workspace(4, 8, ctypes.addressof(n)) == 0
    args = [one, one, one, None, one, one, 4, 8, 1e-5, 0, one, n.value, None]
    for i, bad in ((0, None), (2, None), (4, None), (5, None), (6, -1), (7, 0), (9, 3), (10, None), (11, 0)):
        assert lib.cb200_rms_norm_backward(*(bad if j == i else a for j, a in enumerate(args))) < 0, i

    def heads(data=16, b=512, t=64, h=16, count=4):
        return _HEADS.pack(data, b, t, h, count, 0)

    good = [16, 16, 16, 16, 16, 2, 5, 7, 16, 16, 1e-5, 0, 0, 0, 2, 0]
    for i, bad in ((0, 0), (2, 0), (5, -1), (6, 1 << 32), (8, 0), (9, 15), (9, 18), (12, 4), (13, 1), (14, 3)):
        packed = _QK_ARGS.pack(*(bad if j == i else a for j, a in enumerate(good)))
        assert lib.cb200_qk_norm_rope(heads(), heads(), heads(), heads(), packed, None, None) < 0, i
    packed = _QK_ARGS.pack(*good)
    assert lib.cb200_qk_norm_rope(heads(), heads(), heads(), heads(), _QK_ARGS.pack(*(good[:4] + [0] + good[5:7] + [4] + good[8:])), None, None) == -1
    for view in (heads(data=0), heads(h=8), heads(t=32), heads(b=0), heads(count=3), heads(t=-64)):
        assert lib.cb200_qk_norm_rope(heads(), heads(), heads(), view, packed, None, None) < 0
    for view in (heads(data=0), heads(count=-1), heads(t=-64)):
        assert lib.cb200_qk_norm_rope(heads(), view, heads(), view, packed, None, None) < 0
    assert struct.calcsize("=qqqqii") == 40 and _QK_ARGS.size == 96  # sizeof the C structs
    assert lib.cb200_qk_norm_rope_backward_workspace(16, ctypes.addressof(n)) == 0
    for i, bad in ((6, None), (8, None), (9, None), (10, n.value - 1)):
        args = [heads()] * 6 + [one, one, packed, one, n.value, None, None]
        args[i] = bad
        assert lib.cb200_qk_norm_rope_backward(*args) < 0, i


def test_sizes_that_do_not_fit_32_bits_are_refused():
    import ctypes

    import candle_b200 as cb
    from candle_b200 import _cabi
    from candle_b200.ops import _HEADS, _QK_ARGS

    lib, one, unsupported = _cabi.lib, ctypes.c_void_p(16), -5  # never dereferenced
    n, f32 = ctypes.c_int64(), torch.float32
    for wide in (1 << 29, (1 << 31) - 1):  # the next power of two would count to a negative number
        assert lib.cb200_embedding_scaled(one, one, one, 10, wide, 2, 1.0, 0, 1, None, None) == unsupported
        assert lib.cb200_embedding_backward_workspace(10, wide, 100, ctypes.addressof(n)) == unsupported
        assert lib.cb200_embedding_backward(one, 8, one, one, 10, wide, 100, 1.0, -1, 0, 0, 0, 1, one, 1 << 60, None, None) == unsupported
        assert lib.cb200_rms_norm_backward_workspace(4, wide, ctypes.addressof(n)) == unsupported
        assert lib.cb200_rms_norm_backward(one, one, one, None, one, one, 4, wide, 1e-5, 0, one, 1 << 60, None) == unsupported
        assert lib.cb200_qk_norm_rope_backward_workspace(wide, ctypes.addressof(n)) == unsupported
        for dim, heads in ((wide, 1), (2, wide)):
            h = _HEADS.pack(16, 2 * wide, 2 * wide, dim, heads, 0)
            args = _QK_ARGS.pack(16, 16, 16, 16, 16, 1, 1, 7, dim, 2, 1e-5, 0, 0, 0, 2, 0)
            assert lib.cb200_qk_norm_rope(h, h, h, h, args, None, None) == unsupported
            assert lib.cb200_qk_norm_rope_backward(h, h, h, h, h, h, one, one, args, one, 1 << 60, None, None) == unsupported
    half = _HEADS.pack(16, 1 << 32, 1 << 32, 2, 1 << 30, 0)  # whose sum would be negative
    args = _QK_ARGS.pack(16, 16, 16, 16, 16, 1, 1, 7, 2, 2, 1e-5, 0, 0, 0, 2, 0)
    assert lib.cb200_qk_norm_rope(half, half, half, half, args, None, None) == unsupported

    def meta(*shape, dtype=f32):
        return torch.empty(shape, dtype=dtype, device="meta")

    ids = meta(2, dtype=torch.int64)
    for wide in (1 << 29, (1 << 32) + 8):  # the second is 8 in 32 bits
        with pytest.raises(cb.CandleError, match=str(wide)):
            cb.embedding_scaled(meta(3, wide), ids, 2.0)
        with pytest.raises(cb.CandleError, match=str(wide)):
            cb.embedding_backward(meta(2, wide), ids, 10)
        with pytest.raises(cb.CandleError, match=str(wide)):
            cb.rms_norm_backward(meta(2, wide), meta(2, wide), meta(wide), 1e-5)
        for dim, heads in ((wide, 1), (2, wide)):
            q, k, w, c = meta(1, heads, dim), meta(1, 1, dim), meta(dim), meta(1, 1)
            with pytest.raises(cb.CandleError, match=str(wide)):
                cb.qk_norm_rope(q, k, w, w, 1e-5, c, c)
            with pytest.raises(cb.CandleError, match=str(wide)):
                cb.qk_norm_rope_backward(q, k, q, k, w, w, 1e-5, c, c)


def test_workspaces_grow_with_the_call():
    import ctypes

    from candle_b200 import _cabi

    n = ctypes.c_int64()

    def size(name, *args):
        assert getattr(_cabi.lib, name)(*args, ctypes.addressof(n)) == 0
        return n.value

    # a line of f32 partial sums per row at most, and 8 bytes per row that is too long for one pass
    for rows, cols in ((1, 8), (1, 16384), (1, 1 << 20), (3, 8192), (7, 8193), (2, (1 << 29) - 1)):
        assert rows * cols * 4 <= size("cb200_rms_norm_backward_workspace", rows, cols) <= rows * (cols * 4 + 8) + 16, (rows, cols)
    many = size("cb200_rms_norm_backward_workspace", 1 << 20, 256)
    assert many == size("cb200_rms_norm_backward_workspace", 1 << 21, 256)  # no more lines than the GPU runs CTAs
    assert size("cb200_rms_norm_backward_workspace", 1 << 20, 8193) - size("cb200_rms_norm_backward_workspace", 1 << 20, 8192) >= 8 << 20
    # sorted ids and positions twice, five bytes per row of the table, the long runs; an f32 row per 32 ids above 1024 ids
    for vocab, hidden, ids in ((10, 8, 1), (1000, 8192, 1024), (10, 1 << 20, 64), (100, 64, 8192)):
        sums = ids // 32 * hidden * 4 if ids > 1024 else 0
        least = 16 * ids + 5 * vocab + sums
        assert least <= size("cb200_embedding_backward_workspace", vocab, hidden, ids) <= least + ids // 8 + 10 * 16, (vocab, hidden, ids)


def test_a_padding_id_is_a_row_of_the_table():
    import ctypes

    import candle_b200 as cb
    from candle_b200 import _cabi

    grad, ids = torch.zeros(3, 8), torch.tensor([1, -1, 2])
    for padding in (-100, -1, 10, 1 << 40):  # of ids outside the table every one is reported, so none can be padding
        with pytest.raises(cb.CandleError, match="padding_id"):
            cb.embedding_backward(grad, ids, 10, padding_id=padding)
    with pytest.raises(cb.CandleError, match="no CPU fallback"):
        cb.embedding_backward(grad, ids, 10, padding_id=9)
    one, n = ctypes.c_void_p(16), ctypes.c_int64()
    assert _cabi.lib.cb200_embedding_backward_workspace(10, 8, 100, ctypes.addressof(n)) == 0
    for padding in (-2, 10):
        assert _cabi.lib.cb200_embedding_backward(one, 8, one, one, 10, 8, 100, 1.0, padding, 0, 0, 0, 1, one, n.value, None, None) == -1


def test_cpp_mirror_compiles_and_refuses(tmp_path):
    import os
    import shutil
    import subprocess

    import candle_b200  # noqa: F401  (makes sure the library is built)

    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no g++")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    lib_dir, exe = os.path.join(root, "candle_b200", "_lib"), str(tmp_path / "training_checks")
    subprocess.run([gxx, "-std=c++17", "-Wall", "-Wextra", "-Werror", "-I", os.path.join(root, "include"), "-o", exe,
                    os.path.join(root, "tests", "cpp", "training_checks.cpp"), "-L", lib_dir, "-l:libcandle_b200.so",
                    f"-Wl,-rpath,{lib_dir}"], check=True)
    out = subprocess.run([exe], capture_output=True, text=True)
    lines = out.stdout.strip().splitlines()
    assert out.returncode == 0 and len(lines) == 11 and all(line.startswith("ok ") for line in lines), out.stdout + out.stderr


def test_modules_pass_their_arguments_on(monkeypatch):
    from candle_b200 import nn, ops

    seen = []
    monkeypatch.setattr(ops, "embedding_scaled", lambda *a, **k: seen.append(("scaled", a[2], k)))
    monkeypatch.setattr(ops, "embedding_backward", lambda *a, **k: seen.append(("backward", a[2], k["scale"])))
    monkeypatch.setattr(ops, "rms_norm_backward", lambda *a, **k: seen.append(("norm", a[3], k["grad_sum"])))
    e, n, ids = nn.Embedding(torch.zeros(10, 8), 8), nn.RmsNorm(torch.ones(8), 1e-5), torch.zeros(3, dtype=torch.int64)
    e.forward(ids, scale=2.0, check=False)
    e.backward(torch.zeros(3, 8), ids, scale=2.0)
    n.backward(torch.zeros(3, 8), torch.zeros(3, 8))
    assert seen == [("scaled", 2.0, {"check": False}), ("backward", 10, 2.0), ("norm", 1e-5, None)]


# ---- scaled lookup -----------------------------------------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab,hidden,n,id_dtype", [(50, 64, 1, torch.int64), (300, 1000, 77, torch.uint32), (1000, 4096, 515, torch.int32),
                                                     (200, 7, 33, torch.uint8), (3, 1, 5, torch.int64), (90, 8192, 3, torch.int64),
                                                     (40, 36, 2000, torch.int64), (1000, 520, 20000, torch.uint32)])
def test_scaled_lookup(cb, dtype, vocab, hidden, n, id_dtype):
    table = rand(1, (vocab, hidden), DTYPES[dtype])
    ids = make_ids(2, n, vocab, "uniform", id_dtype)
    scale = math.sqrt(hidden)
    y = cb.embedding_scaled(table, ids, scale)
    # one product in f32, one rounding: the same as torch's f32 product rounded
    want = (table[as_long(ids)].float() * torch.tensor(scale, dtype=torch.float32)).to(DTYPES[dtype])
    assert torch.equal(y, want)
    check(y, table[as_long(ids)].double() * scale, 2 * U * table[as_long(ids)].double().abs() * scale)


@pytest.mark.gpu
def test_scaled_lookup_shapes_alignment_and_bad_ids(cb):
    base = rand(3, (101 * 24 + 1,), torch.bfloat16)
    for table in (base[:101 * 24].view(101, 24), base[1:].view(101, 24)):  # 16-byte aligned, 2-byte aligned
        ids = make_ids(4, 30, 101, "uniform").view(5, 6)
        out = torch.empty(5 * 6 * 24 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(5, 6, 24)
        y = cb.embedding_scaled(table, ids, 1.5, out=out)
        assert y is out and torch.equal(y, (table[ids].float() * 1.5).bfloat16())
    assert cb.embedding_scaled(table, ids[:0], 2.0).shape == (0, 6, 24)
    bad = ids.clone()
    bad[1, 2] = 101
    out.fill_(7.0)
    with pytest.raises(cb.InvalidIndex):
        cb.embedding_scaled(table, bad, 1.5, out=out)
    want = (table[bad.clamp(max=100)].float() * 1.5).bfloat16()
    want[1, 2] = 7.0
    assert torch.equal(out, want)
    with pytest.raises(cb.InvalidIndex):
        cb.embedding_scaled(table, torch.tensor([-1], device="cuda"), 1.0)
    with pytest.raises(cb.CandleError, match="overlaps"):
        cb.embedding_scaled(table, ids[0, :1], 2.0, out=table[3:4])


# ---- the table's gradient ----------------------------------------------------------------------------------


def table_grad_64(grad, ids, vocab, scale, padding=None):
    ids = as_long(ids).reshape(-1)
    g = grad.reshape(-1, grad.shape[-1]).double()
    if padding is not None:
        keep = ids != padding
        ids, g = ids[keep], g[keep]
    total = torch.zeros(vocab, g.shape[1], dtype=torch.float64, device=g.device).index_add_(0, ids, g)
    sizes = torch.zeros(vocab, g.shape[1], dtype=torch.float64, device=g.device).index_add_(0, ids, g.abs())
    count = torch.bincount(ids, minlength=vocab).double()[:, None]
    return total * scale, sizes * scale, count


GRAD_CASES = [
    # n, vocab, hidden: no token to many; one id, digits of the sort at their edges; odd columns
    (0, 10, 8), (1, 1, 1), (1, 1000, 64), (2, 2, 33), (63, 3, 16), (64, 1, 40), (65, 513, 100), (127, 511, 64), (128, 512, 24),
    (129, 4, 257), (1000, 300, 1000), (4095, 262143, 8), (4096, 5000, 64), (4097, 262144, 16), (20000, 700, 136), (70001, 1200, 72),
]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["uniform", "same", "skew", "falling"])
@pytest.mark.parametrize("n,vocab,hidden", GRAD_CASES)
def test_table_grad_of_whole_numbers_is_exact(cb, n, vocab, hidden, kind):
    # |terms| <= 8, at most 70001 of them: every partial sum is a whole number below 2^24
    g = torch.Generator().manual_seed(n + vocab)
    grad = torch.randint(-8, 9, (n, hidden), generator=g).cuda()
    ids = make_ids(n, n, vocab, kind)
    want = torch.zeros(vocab, hidden, dtype=torch.int64, device="cuda").index_add_(0, ids, grad)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        got = cb.embedding_backward(grad.to(dtype), ids, vocab, out_dtype=torch.float32)
        assert got.shape == (vocab, hidden) and torch.equal(got.double(), want.double()), dtype
        before = torch.randint(-8, 9, (vocab, hidden), generator=g).cuda()
        acc = before.float()
        assert cb.embedding_backward(grad.to(dtype), ids, vocab, scale=2.0, out=acc, accumulate=True) is acc
        assert torch.equal(acc.double(), (before + 2 * want).double()), dtype


@pytest.mark.gpu
@pytest.mark.parametrize("n,vocab,hidden,kind", [
    (1024, 50, 72, "skew"), (1025, 50, 72, "skew"), (8192, 90, 72, "skew"), (8193, 90, 72, "skew"),  # where the launches change
    (9000, 262145, 24, "uniform"), (20000, (1 << 27) + 3, 1, "skew"),  # three and four digits
    (40000, 300, 4096, "uniform"), (40000, 300, 4096, "skew"), (60000, 200, 2056, "skew"),  # many long runs, several vectors per lane
    (30000, 30000, 4096, "uniform"), (9000, 9, 515, "falling"),
])
def test_table_grad_over_the_kernels_of_larger_batches(cb, n, vocab, hidden, kind):
    # whole numbers of at most 8: exact, as above
    g = torch.Generator(device="cuda").manual_seed(n)
    grad = torch.randint(-8, 9, (n, hidden), generator=g, device="cuda", dtype=torch.int32)
    ids = make_ids(n + 1, n, vocab, kind)
    for dtype, wide in ((torch.bfloat16, False), (torch.bfloat16, True), (torch.float32, True)):
        if not wide and vocab * hidden > 1 << 27:
            continue
        out_dtype = torch.float32 if wide else dtype
        got = cb.embedding_backward(grad.to(dtype), ids, vocab, out_dtype=out_dtype)
        want = torch.zeros(vocab, hidden, dtype=torch.float32, device="cuda").index_add_(0, ids, grad.float())
        assert torch.equal(got, want.to(out_dtype))
        acc = torch.full((vocab, hidden), 2.0, dtype=out_dtype, device="cuda")
        cb.embedding_backward(grad.to(dtype), ids, vocab, scale=0.5, out=acc, accumulate=True)
        assert torch.equal(acc, (2.0 + 0.5 * want).to(out_dtype))
        del got, want, acc


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("n,vocab,hidden,kind,id_dtype", [(1, 100, 64, "uniform", torch.int64), (513, 100, 1000, "skew", torch.uint32),
                                                          (3000, 2000, 136, "uniform", torch.int32), (5000, 200, 65, "skew", torch.uint8),
                                                          (9000, 40, 4096, "skew", torch.int64)])
def test_table_grad(cb, dtype, wide, n, vocab, hidden, kind, id_dtype):
    grad = rand(5, (n, hidden), DTYPES[dtype])
    ids = make_ids(6, n, vocab, kind, id_dtype)
    out_dtype = torch.float32 if wide else DTYPES[dtype]
    got = cb.embedding_backward(grad, ids, vocab, scale=math.sqrt(hidden), out_dtype=out_dtype)
    want, sizes, count = table_grad_64(grad, ids, vocab, math.sqrt(hidden))
    assert got.dtype == out_dtype
    # at most 64 tokens in a row, then 9000 / 64 chunk sums over eight warps, then the warps: fewer than 128 steps; 2 for the scale
    depth = count.clamp(max=128) + 2
    check(got, want, depth * U * sizes)
    assert not torch.signbit(got[count[:, 0] == 0]).any()  # rows without tokens are +0
    again = cb.embedding_backward(grad, ids, vocab, scale=math.sqrt(hidden), out_dtype=out_dtype)
    assert torch.equal(got, again)
    before = rand(7, (vocab, hidden), out_dtype)
    acc = cb.embedding_backward(grad, ids, vocab, scale=math.sqrt(hidden), out=before.clone(), accumulate=True)
    check(acc, want + before.double(), (depth + 2) * U * (sizes + before.double().abs()))
    assert torch.equal(acc[count[:, 0] == 0], before[count[:, 0] == 0])


@pytest.mark.gpu
def test_table_grad_strides_padding_and_bad_ids(cb):
    vocab, hidden = 70, 48
    wide = rand(8, (6, 50, 96), torch.bfloat16)
    ids = make_ids(9, 300, vocab, "skew").view(6, 50)
    for grad in (wide[..., :48], wide[..., 8:56], wide[..., 3:51]):  # rows 96 apart; the last is not 16-byte aligned
        want = table_grad_64(grad, ids, vocab, 1.0)
        check(cb.embedding_backward(grad, ids, vocab), want[0], 130 * U * want[1])
    one = rand(10, (1, hidden), torch.float32).expand(300, hidden)  # one row for all tokens
    want = table_grad_64(one, ids.view(-1), vocab, 1.0)
    check(cb.embedding_backward(one, ids.view(-1), vocab), want[0], 130 * U * want[1])
    hot = int(torch.bincount(ids.view(-1)).argmax())
    grad = wide[..., :48]
    want = table_grad_64(grad, ids, vocab, 1.0, padding=hot)
    got = cb.embedding_backward(grad, ids, vocab, padding_id=hot)
    check(got, want[0], 130 * U * want[1])
    assert not got[hot].any()
    bad = ids.clone()
    bad[0, 3], bad[5, 49] = vocab, -7
    status = torch.zeros(4, dtype=torch.int64, device="cuda")
    got = cb.embedding_backward(grad, bad, vocab, check=False, status=status)
    keep = (bad >= 0) & (bad < vocab)
    want = table_grad_64(grad[keep], bad[keep], vocab, 1.0)
    check(got, want[0], 130 * U * want[1])
    assert status[0].item() & 0xFFFFFFFF == 1 and status[3].item() == vocab
    with pytest.raises(cb.InvalidIndex):
        cb.embedding_backward(grad, bad, vocab)
    with pytest.raises(cb.CandleError, match="missing"):
        cb.embedding_backward(grad, ids, vocab, accumulate=True)
    with pytest.raises(cb.CandleError, match="overlaps"):
        big = torch.zeros(vocab + 300, hidden, device="cuda")
        cb.embedding_backward(big[vocab - 1:-1], ids.view(-1), vocab, out=big[:vocab])
    assert cb.embedding_backward(grad, ids, 0, check=False).shape == (0, hidden)
    assert cb.embedding_backward(wide[..., :0], ids, vocab).shape == (vocab, 0)


@pytest.mark.gpu
def test_table_grad_infinities_and_nan_stay_in_their_rows(cb):
    grad, ids = rand(11, (500, 32), torch.float32), make_ids(12, 500, 20, "uniform")
    grad[17, 3], grad[99, 5] = math.inf, math.nan
    got = cb.embedding_backward(grad, ids, 20)
    where = torch.zeros(20, 32, dtype=torch.bool, device="cuda")
    where[ids[17], 3] = where[ids[99], 5] = True
    assert torch.equal(~torch.isfinite(got), where)


# ---- gradient of the RMS norm ------------------------------------------------------------------------------


def norm_grad_64(grad, x, w, eps):
    """The formula's gradient and the sizes of its terms; rows over the last dimension."""
    g, x, w = grad.double(), x.double(), w.double()
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    unit, gw = x * r, g * w
    dx = r * (gw - unit * (gw * unit).mean(-1, keepdim=True))
    size = r * (gw.abs() + unit.abs() * (gw * unit).abs().mean(-1, keepdim=True))
    terms = (g * unit).reshape(-1, x.shape[-1])
    return dx, size, terms.sum(0), terms.abs().sum(0)


NORM_SHAPES = [(600, 3348), (50, 6150), (7, 12000), (400, 4097), (333, 130), (1, 1), (1, 8), (3, 7), (5, 64), (2, 128), (300, 96), (1000, 768), (33, 1000), (64, 2048), (9, 4096), (700, 4096), (1200, 8192),
               (2, 8192), (5, 10000), (3, 16384), (40, 257), (20000, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", NORM_SHAPES)
def test_rms_norm_backward(cb, dtype, rows, cols):
    t, eps = DTYPES[dtype], 1e-5
    x, grad, w = rand(1, (rows, cols), t), rand(2, (rows, cols), t), rand(3, (cols,), t, 1.0, 0.1)
    extra = rand(4, (rows, cols), t)
    dx, size, dw, dw_size = norm_grad_64(grad, x, w, eps)
    steps = 2 * SUM(cols) + OPS
    got, got_w = cb.rms_norm_backward(grad, x, w, eps)
    check(got, dx, steps * U * size)
    # rows per accumulator (the GPU holds at least 148), then at most 2 * 148 partial sums over eight warps
    check(got_w, dw, (rows / 148 + 2 * 148 / 8 + 8 + SUM(cols) + OPS) * U * dw_size)
    again, again_w = cb.rms_norm_backward(grad, x, w, eps)
    assert torch.equal(got, again) and torch.equal(got_w, again_w)
    summed, _ = cb.rms_norm_backward(grad, x, w, eps, grad_sum=extra)
    check(summed, dx + extra.double(), (steps + 1) * U * (size + extra.double().abs()))
    for which in range(3):  # in place
        args = [grad.clone(), x.clone(), extra.clone()]
        in_place, w_too = cb.rms_norm_backward(args[0], args[1], w, eps, grad_sum=args[2], out=args[which])
        assert in_place is args[which] and torch.equal(in_place, summed) and torch.equal(w_too, got_w)


@pytest.mark.gpu
def test_rms_norm_backward_odd_rows_and_refusals(cb):
    t = torch.bfloat16
    for rows, cols in ((40, 512), (12, 8192)):
        x, grad, w = rand(1, (rows, cols), t), rand(2, (rows, cols), t), rand(3, (cols,), t, 1.0, 0.1)
        base = [torch.empty(rows * cols + 1, dtype=t, device="cuda") for _ in range(2)]  # not 16-byte aligned
        xs, gs = base[0][1:].view(rows, cols).copy_(x), base[1][1:].view(rows, cols).copy_(grad)
        dx, size, dw, dw_size = norm_grad_64(grad, x, w, 1e-5)
        for a, b in ((gs, x), (grad, xs), (gs, xs)):
            got, got_w = cb.rms_norm_backward(a, b, w, 1e-5)
            check(got, dx, (2 * SUM(cols) + OPS) * U * size)
            check(got_w, dw, (60 + SUM(cols) + OPS) * U * dw_size)
        # rows of zeros, of huge values, with infinities and NaN: only they are touched, and they poison the weights' gradient alone
        x[1] = 0
        x[2] *= 1e4
        dx, size, dw, dw_size = norm_grad_64(grad, x, w, 1e-5)
        got, got_w = cb.rms_norm_backward(grad, x, w, 1e-5)
        check(got, dx, (2 * SUM(cols) + OPS) * U * size)
        check(got_w, dw, (60 + SUM(cols) + OPS) * U * dw_size)
        x[3, 5], grad[4, 6] = math.inf, math.nan
        clean = torch.arange(rows, device="cuda") % rows
        clean = clean[(clean != 3) & (clean != 4)]
        got, _ = cb.rms_norm_backward(grad, x, w, 1e-5)
        check(got[clean], dx[clean], ((2 * SUM(cols) + OPS) * U * size)[clean])
    empty, ew = cb.rms_norm_backward(grad[:0], x[:0], w, 1e-5)
    assert empty.shape == (0, cols) and not ew.any()
    three = rand(5, (2, 3, 512), torch.float32)
    dx, _ = cb.rms_norm_backward(three, three, torch.ones(512, device="cuda"), 1e-5)
    assert dx.shape == three.shape
    buf = torch.zeros(5, 512, device="cuda")
    with pytest.raises(cb.CandleError, match="overlaps"):
        cb.rms_norm_backward(buf[:4], buf[:4].clone(), torch.ones(512, device="cuda"), 1e-5, out=buf[1:])


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", [(2, 1 << 20), (1, 300001), (300, 9000)])
def test_rms_norm_backward_of_very_long_rows(cb, rows, cols):
    x, grad, w = rand(1, (rows, cols), torch.float32), rand(2, (rows, cols), torch.float32), rand(3, (cols,), torch.float32, 1.0, 0.1)
    dx, size, dw, dw_size = norm_grad_64(grad, x, w, 1e-5)
    got, got_w = cb.rms_norm_backward(grad, x, w, 1e-5)
    check(got, dx, (2 * SUM(cols) + OPS) * U * size)
    check(got_w, dw, (rows + SUM(cols) + OPS) * U * dw_size)


@pytest.mark.gpu
def test_nothing_behind_the_workspace_is_written(cb):
    import ctypes

    from candle_b200 import _cabi

    tail, stream, n = 1 << 20, torch.cuda.current_stream().cuda_stream, ctypes.c_int64()

    def workspace(name, *args):
        assert getattr(_cabi.lib, name)(*args, ctypes.addressof(n)) == 0
        return torch.full((n.value + tail,), 0xA5, dtype=torch.uint8, device="cuda"), n.value

    # the smallest calls, both sides of the sizes where scratch changes, and lengths for every route
    for rows, cols in ((1, 8), (1, 9), (5, 64), (600, 8192), (2, 8191), (3, 8193), (700, 8193), (1, 50000), (3000, 264)):
        x, grad, w = rand(1, (rows, cols), torch.float32), rand(2, (rows, cols), torch.float32), rand(3, (cols,), torch.float32)
        ws, size = workspace("cb200_rms_norm_backward_workspace", rows, cols)
        dx, dw = torch.empty_like(x), torch.empty(cols, device="cuda")
        _cabi.call("cb200_rms_norm_backward", grad.data_ptr(), x.data_ptr(), w.data_ptr(), None, dx.data_ptr(), dw.data_ptr(), rows, cols,
                   1e-5, 0, ws.data_ptr(), size, stream)
        want, want_w = cb.rms_norm_backward(grad, x, w, 1e-5)
        assert torch.equal(dx, want) and torch.equal(dw, want_w) and (ws[size:] == 0xA5).all(), (rows, cols)
    for ids, vocab, hidden in ((1, 1, 8), (64, 3, 65), (1024, 5, 24), (1025, 5, 24), (8192, 70, 8), (8193, 70, 8), (40000, 1 << 19, 8)):
        grad, which = rand(4, (ids, hidden), torch.float32), make_ids(5, ids, vocab, "skew")
        ws, size = workspace("cb200_embedding_backward_workspace", vocab, hidden, ids)
        out = torch.empty(vocab, hidden, device="cuda")
        _cabi.call("cb200_embedding_backward", grad.data_ptr(), hidden, which.data_ptr(), out.data_ptr(), vocab, hidden, ids, 1.0, -1, 0, 0, 0, 2,
                   ws.data_ptr(), size, None, stream)
        assert torch.equal(out, cb.embedding_backward(grad, which, vocab)) and (ws[size:] == 0xA5).all(), (ids, vocab, hidden)


# ---- head norms with rotation ------------------------------------------------------------------------------


def turn_64(x, cos, sin, interleaved, sign=1.0):
    """(rotated, sizes of the terms): the first 2 * cos.shape[-1] columns of x in 64 bits."""
    half = cos.shape[-1]
    i1 = torch.arange(half, device=x.device) * 2 if interleaved else torch.arange(half, device=x.device)
    i2 = i1 + 1 if interleaved else i1 + half
    y, size = x.clone(), x.abs()
    a, b, s = x[..., i1], x[..., i2], sin * sign
    y[..., i1], y[..., i2] = a * cos - b * s, a * s + b * cos
    size[..., i1], size[..., i2] = (a * cos).abs() + (b * s).abs(), (a * s).abs() + (b * cos).abs()
    return y, size


def angles_64(cos, sin, positions, tokens_shape):
    if positions is None:
        positions = torch.arange(tokens_shape[-1], device=cos.device).expand(tokens_shape)
    positions = as_long(positions)
    return cos.double()[positions].unsqueeze(-2), sin.double()[positions].unsqueeze(-2)


def heads_64(x, w, eps, c, s, interleaved):
    f = x.double()
    u = f * (f.square().mean(-1, keepdim=True) + eps).rsqrt() * w.double()
    return turn_64(u, c, s, interleaved)


def heads_grad_64(grad, x, w, eps, c, s, interleaved):
    v, size_v = turn_64(grad.double(), c, s, interleaved, -1.0)
    dx, _, dw, _ = norm_grad_64(v, x, w, eps)
    _, size, _, dw_size = norm_grad_64(size_v, x.double().abs(), w.double().abs(), eps)
    return dx, size, dw, dw_size


def qkv_views(layout, batch, length, hq, hk, d, t, seed):
    """q and k in the given memory layout, seen as [b, t, h, d] (or [t, h, d])."""
    if layout == "packed":
        qkv = rand(seed, (batch, length, hq + 2 * hk, d), t)
        return qkv[:, :, :hq], qkv[:, :, hq:hq + hk]
    if layout == "head-major":
        return rand(seed, (batch, hq, length, d), t).transpose(1, 2), rand(seed + 1, (batch, hk, length, d), t).transpose(1, 2)
    if layout == "flat":
        return rand(seed, (batch * length, hq, d), t), rand(seed + 1, (batch * length, hk, d), t)
    if layout == "shifted":  # rows that are not 16-byte aligned
        wide = rand(seed, (batch, length, hq + hk, d + 1), t)
        return wide[:, :, :hq, 1:], wide[:, :, hq:, 1:]
    return rand(seed, (batch, length, hq, d), t), rand(seed + 1, (batch, length, hk, d), t)


HEAD_CASES = [
    # layout, batch, length, q heads, k heads, dim, rotated, interleaved, positions
    ("plain", 1, 1, 1, 1, 2, 2, False, None),
    ("plain", 2, 5, 4, 2, 64, 64, False, None),
    ("packed", 2, 33, 8, 2, 128, 128, False, torch.int64),
    ("packed", 64, 1, 32, 8, 128, 128, False, torch.int64),
    ("head-major", 2, 17, 6, 3, 128, 128, True, None),
    ("flat", 1, 19, 5, 1, 80, 80, False, torch.int32),
    ("packed", 3, 21, 12, 12, 80, 32, True, torch.uint32),
    ("plain", 1, 9, 3, 1, 96, 48, False, None),
    ("plain", 1, 7, 2, 2, 256, 256, False, torch.uint8),
    ("plain", 2, 3, 7, 1, 512, 512, True, None),
    ("plain", 1, 4, 2, 1, 1024, 256, False, None),
    ("plain", 1, 3, 1, 1, 1536, 1536, True, None),
    ("shifted", 2, 11, 4, 2, 64, 64, False, torch.int64),
    ("plain", 2, 11, 3, 5, 66, 30, True, None),
    ("plain", 1, 13, 2, 1, 7, 6, False, None),
    ("plain", 1, 5, 4, 4, 192, 2, True, None),
    ("packed", 1, 700, 16, 4, 64, 64, True, torch.int64),
    ("packed", 2, 1500, 8, 8, 128, 64, False, None),
    ("plain", 4, 6, 3, 0, 64, 64, False, None),
    ("plain", 4, 6, 0, 3, 64, 64, False, torch.int64),
    ("plain", 1, 2050, 9, 1, 72, 72, False, None),
    ("plain", 0, 6, 3, 2, 64, 64, False, torch.int64),
    ("flat", 1, 0, 3, 2, 64, 64, False, None),
]


def head_case(case, dtype, table_dtype, seed=0):
    layout, batch, length, hq, hk, d, rd, interleaved, pos_dtype = case
    t = DTYPES[dtype]
    q, k = qkv_views(layout, batch, length, hq, hk, d, t, 10 + seed)
    wq, wk = rand(20 + seed, (d,), t, 1.0, 0.2), rand(21 + seed, (d,), t, 1.0, 0.2)
    n_pos = length + 60
    angle = torch.arange(n_pos, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, rd, 2, dtype=torch.float64) / rd)
    tt = torch.float32 if table_dtype == "f32" else t
    cos, sin = angle.cos().to(tt).cuda(), angle.sin().to(tt).cuda()
    positions = None
    if pos_dtype is not None:
        g = torch.Generator().manual_seed(30 + seed)
        shape = q.shape[:-2]
        positions = torch.randint(0, min(n_pos, 250), shape, generator=g)
        positions = positions.to(torch.int32).view(torch.uint32).cuda() if pos_dtype == torch.uint32 else positions.to(pos_dtype).cuda()
    return q, k, wq, wk, cos, sin, positions, interleaved


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,table_dtype", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32")])
@pytest.mark.parametrize("case", HEAD_CASES, ids=lambda c: "-".join(map(str, c[:8])))
def test_qk_norm_rope(cb, case, dtype, table_dtype):
    q, k, wq, wk, cos, sin, positions, interleaved = head_case(case, dtype, table_dtype)
    eps = 1e-5
    got = cb.qk_norm_rope(q, k, wq, wk, eps, cos, sin, positions=positions, interleaved=interleaved)
    c, s = angles_64(cos, sin, positions, q.shape[:-2])
    for y, x, w in ((got[0], q, wq), (got[1], k, wk)):
        want, size = heads_64(x, w, eps, c, s, interleaved)
        assert y.shape == x.shape and y.is_contiguous()
        check(y, want, (SUM(x.shape[-1]) / 2 + OPS) * U * size)
    if case[0] == "packed":  # into the projection itself; the values behind the keys stay
        base = q._base.clone()
        hq, hk = q.shape[2], k.shape[2]
        values = base[:, :, hq + hk:].clone()
        iq, ik = base[:, :, :hq], base[:, :, hq:hq + hk]
        out = cb.qk_norm_rope(iq, ik, wq, wk, eps, cos, sin, positions=positions, interleaved=interleaved, out=(iq, ik))
        assert out[0] is iq and torch.equal(iq, got[0]) and torch.equal(ik, got[1]) and torch.equal(base[:, :, hq + hk:], values)
    elif case[0] == "head-major":
        outs = tuple(torch.empty_like(x.transpose(1, 2)).transpose(1, 2) for x in (q, k))
        cb.qk_norm_rope(q, k, wq, wk, eps, cos, sin, positions=positions, interleaved=interleaved, out=outs)
        assert torch.equal(outs[0], got[0]) and torch.equal(outs[1], got[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,table_dtype", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32")])
@pytest.mark.parametrize("case", HEAD_CASES, ids=lambda c: "-".join(map(str, c[:8])))
def test_qk_norm_rope_backward(cb, case, dtype, table_dtype):
    q, k, wq, wk, cos, sin, positions, interleaved = head_case(case, dtype, table_dtype)
    eps = 1e-5
    gq, gk = rand(40, q.shape, q.dtype), rand(41, k.shape, k.dtype)
    run = lambda **kw: cb.qk_norm_rope_backward(gq, gk, q, k, wq, wk, eps, cos, sin, positions=positions, interleaved=interleaved, **kw)  # noqa: E731
    got = run()
    c, s = angles_64(cos, sin, positions, q.shape[:-2])
    for dx, dw, g, x, w in ((got[0], got[2], gq, q, wq), (got[1], got[3], gk, k, wk)):
        want, size, want_w, size_w = heads_grad_64(g, x, w, eps, c, s, interleaved)
        d = x.shape[-1]
        check(dx, want, (2 * SUM(d) + OPS) * U * size)
        # rows per accumulator and its partial sums: at most 4736 lines over eight warps when every warp keeps one
        rows = x.numel() // d
        check(dw, want_w, (min(rows, 4736) / 8 + rows / 148 + 8 + SUM(d) / 2 + OPS) * U * size_w)
    again = run()
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    gq2, gk2 = gq.clone(), gk.clone()
    in_place = cb.qk_norm_rope_backward(gq2, gk2, q, k, wq, wk, eps, cos, sin, positions=positions, interleaved=interleaved, out=(gq2, gk2))
    assert all(torch.equal(a, b) for a, b in zip(got, in_place))
    if case[0] == "packed":  # the gradient of the projection's q and k parts
        base = torch.full_like(q._base, 3.0)
        hq, hk = q.shape[2], k.shape[2]
        run(out=(base[:, :, :hq], base[:, :, hq:hq + hk]))
        assert torch.equal(base[:, :, :hq], got[0]) and torch.equal(base[:, :, hq:hq + hk], got[1]) and (base[:, :, hq + hk:] == 3.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("d,rd", [(128, 128), (64, 32), (66, 30)])
def test_qk_norm_rope_bad_positions_zero_rows_and_nan(cb, d, rd):
    case = ("packed", 3, 40, 4, 2, d, rd, False, torch.int64)
    q, k, wq, wk, cos, sin, positions, _ = head_case(case, "bf16", "f32")
    q[0, 1, 2] = 0
    q[0, 2, 1, 5], k[1, 3, 1, 0] = math.nan, math.inf
    c, s = angles_64(cos, sin, positions, q.shape[:-2])
    got = cb.qk_norm_rope(q, k, wq, wk, 1e-5, cos, sin, positions=positions)
    assert not got[0][0, 1, 2].any()
    for y, x, w, bad in ((got[0], q, wq, (0, 2, 1)), (got[1], k, wk, (1, 3, 1))):
        want, size = heads_64(x, w, 1e-5, c, s, False)
        ok = torch.ones(x.shape[:-1], dtype=torch.bool, device="cuda")
        ok[bad] = False
        check(y[ok], want[ok], ((SUM(d) / 2 + OPS) * U * size)[ok])
        assert torch.isnan(y[bad]).any()
    # tokens at positions that the tables do not have
    q, k, wq, wk, cos, sin, positions, _ = head_case(case, "bf16", "f32")
    full = cb.qk_norm_rope(q, k, wq, wk, 1e-5, cos, sin, positions=positions)
    wrong = positions.clone()
    wrong[0, 0], wrong[2, 39] = cos.shape[0], -1
    outs = (torch.full_like(q, 9.0).contiguous(), torch.full_like(k, 9.0).contiguous())
    with pytest.raises(cb.InvalidIndex):
        cb.qk_norm_rope(q, k, wq, wk, 1e-5, cos, sin, positions=wrong, out=outs)
    ok = wrong == positions
    for y, f in zip(outs, full):
        assert torch.equal(y[ok], f[ok]) and (y[~ok] == 9.0).all()
    gq, gk = rand(40, q.shape, q.dtype), rand(41, k.shape, k.dtype)
    status = torch.zeros(4, dtype=torch.int64, device="cuda")
    outs = (torch.full_like(q, 9.0).contiguous(), torch.full_like(k, 9.0).contiguous())
    got = cb.qk_norm_rope_backward(gq, gk, q, k, wq, wk, 1e-5, cos, sin, positions=wrong, out=outs, check=False, status=status)
    assert status[0].item() & 0xFFFFFFFF == 1
    gq[~ok], gk[~ok] = 0, 0
    c, s = angles_64(cos, sin, positions, q.shape[:-2])
    for dx, dw, g, x, w in ((got[0], got[2], gq, q, wq), (got[1], got[3], gk, k, wk)):
        want, size, want_w, size_w = heads_grad_64(g, x, w, 1e-5, c, s, False)
        check(dx[ok], want[ok], ((2 * SUM(d) + OPS) * U * size)[ok])
        assert (dx[~ok] == 9.0).all()
        check(dw, want_w, (120 + SUM(d) / 2 + OPS) * U * size_w)
    with pytest.raises(cb.InvalidIndex):
        cb.qk_norm_rope_backward(gq, gk, q, k, wq, wk, 1e-5, cos, sin, positions=wrong)
    with pytest.raises(cb.CandleError, match="overlaps"):
        cb.qk_norm_rope(q, k, wq, wk, 1e-5, cos, sin, positions=positions, out=(q._base[:, :, 1:5], k))
    row = torch.empty(3, 40, 1, d, dtype=q.dtype, device="cuda").expand(q.shape)
    with pytest.raises(RuntimeError, match="rows overlap"):
        cb.qk_norm_rope(q, k, wq, wk, 1e-5, cos, sin, positions=positions, out=(row, torch.empty_like(k)))


@pytest.mark.gpu
def test_head_norms_of_broadcast_inputs(cb):
    # one row for all heads and tokens, read through strides of zero; the gradient is that of every use
    d = 64
    q = rand(1, (d,), torch.float32).expand(2, 9, 4, d)
    k = rand(2, (2, 1, 1, d), torch.float32).expand(2, 9, 2, d)
    w, cos = torch.ones(d, device="cuda"), torch.rand(9, d // 2, device="cuda")
    sin = (1 - cos * cos).sqrt()
    dense = cb.qk_norm_rope(q.contiguous(), k.contiguous(), w, w, 1e-6, cos, sin)
    assert all(torch.equal(a, b) for a, b in zip(cb.qk_norm_rope(q, k, w, w, 1e-6, cos, sin), dense))
    g = (rand(3, (1, 1, 1, d), torch.float32).expand(2, 9, 4, d), rand(4, (2, 9, 1, d), torch.float32).expand(2, 9, 2, d))
    dense = cb.qk_norm_rope_backward(g[0].contiguous(), g[1].contiguous(), q.contiguous(), k.contiguous(), w, w, 1e-6, cos, sin)
    assert all(torch.equal(a, b) for a, b in zip(cb.qk_norm_rope_backward(*g, q, k, w, w, 1e-6, cos, sin), dense))


# ---- gradients against differences, and the operators together ---------------------------------------------


@pytest.mark.gpu
def test_gradients_against_differences(cb):
    """Directional derivatives of the 64-bit statements by central differences (step 1e-5: off by about 1e-9 of the terms)
    against the operators' gradients in f32 (off by at most a few hundred U of the terms)."""
    torch.manual_seed(0)
    h, tol = 1e-5, 500 * U
    x, w = rand(1, (6, 96), torch.float32), rand(2, (96,), torch.float32, 1.0, 0.2)
    g, ex, ew = rand(3, (6, 96), torch.float32), rand(4, (6, 96), torch.float64), rand(5, (96,), torch.float64)
    f = lambda a, b: (a * (a.square().mean(-1, keepdim=True) + 1e-5).rsqrt() * b * g.double()).sum()  # noqa: E731
    dx, dw = cb.rms_norm_backward(g, x, w, 1e-5)
    X, W = x.double(), w.double()
    for got, e, diff in ((dx, ex, f(X + h * ex, W) - f(X - h * ex, W)), (dw, ew, f(X, W + h * ew) - f(X, W - h * ew))):
        terms = (got.double() * e).abs().sum()
        assert abs((got.double() * e).sum() - diff / (2 * h)) <= tol * terms
    for interleaved in (False, True):
        q, k = rand(6, (5, 3, 32), torch.float32), rand(7, (5, 2, 32), torch.float32)
        wq, wk = rand(8, (32,), torch.float32, 1.0, 0.2), rand(9, (32,), torch.float32, 1.0, 0.2)
        ang = rand(10, (20, 10), torch.float64) * 3
        cos, sin, pos = ang.cos().float(), ang.sin().float(), torch.tensor([3, 19, 0, 7, 7], device="cuda")
        gq, gk = rand(11, q.shape, q.dtype), rand(12, k.shape, k.dtype)
        c, s = angles_64(cos, sin, pos, (5,))
        loss = lambda a, b, u, v: ((heads_64(a, u, 1e-5, c, s, interleaved)[0] * gq.double()).sum()  # noqa: E731
                                   + (heads_64(b, v, 1e-5, c, s, interleaved)[0] * gk.double()).sum())
        got = cb.qk_norm_rope_backward(gq, gk, q, k, wq, wk, 1e-5, cos, sin, positions=pos, interleaved=interleaved)
        at = [t.double() for t in (q, k, wq, wk)]
        for i, t in enumerate(at):
            e = rand(13 + i, t.shape, torch.float64)
            up, down = list(at), list(at)
            up[i], down[i] = t + h * e, t - h * e
            slope = (loss(*up) - loss(*down)) / (2 * h)
            assert abs((got[i].double() * e).sum() - slope) <= tol * (got[i].double() * e).abs().sum()


def block_step(cb, p, ids, g_out):
    """One training step's path: scaled lookup, residual norm, projection, head norms with rotation, and back."""
    hq, hk, d, eps = 4, 2, 64, 1e-5
    scale = math.sqrt(p["table"].shape[1])
    e = cb.embedding_scaled(p["table"], ids, scale, check=False)
    y, h = cb.rms_norm(e, p["alpha"], eps, residual=p["res"], return_sum=True)
    qkv = (y @ p["proj"]).view(*ids.shape, hq + hk, d)
    q, k = qkv[..., :hq, :], qkv[..., hq:, :]
    oq, ok = cb.qk_norm_rope(q, k, p["wq"], p["wk"], eps, p["cos"], p["sin"])
    d_qkv = torch.empty_like(qkv)
    _, _, dwq, dwk = cb.qk_norm_rope_backward(g_out[0], g_out[1], q, k, p["wq"], p["wk"], eps, p["cos"], p["sin"],
                                              out=(d_qkv[..., :hq, :], d_qkv[..., hq:, :]))
    d_qkv = d_qkv.view(*ids.shape, -1)
    dy = d_qkv @ p["proj"].t()
    dproj = y.flatten(0, 1).t() @ d_qkv.flatten(0, 1)
    dh, dalpha = cb.rms_norm_backward(dy, h, p["alpha"], eps, grad_sum=g_out[2])
    dtable = cb.embedding_backward(dh, ids, p["table"].shape[0], scale=scale, check=False)
    return oq, ok, h, dwq, dwk, dproj, dalpha, dh, dtable


def block_inputs(dtype, seed, b=3, t=37):
    vocab, hidden, hq, hk, d = 120, 256, 4, 2, 64
    p = {"table": rand(seed, (vocab, hidden), dtype, std=0.1), "alpha": rand(seed + 1, (hidden,), dtype, 1.0, 0.1),
         "res": rand(seed + 2, (b, t, hidden), dtype), "proj": rand(seed + 3, (hidden, (hq + hk) * d), dtype, std=1 / 16),
         "wq": rand(seed + 4, (d,), dtype, 1.0, 0.1), "wk": rand(seed + 5, (d,), dtype, 1.0, 0.1)}
    ang = torch.arange(t, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    p["cos"], p["sin"] = ang.cos().to(dtype).cuda(), ang.sin().to(dtype).cuda()
    ids = make_ids(seed + 6, b * t, vocab, "skew").view(b, t)
    g = (rand(seed + 7, (b, t, hq, d), dtype), rand(seed + 8, (b, t, hk, d), dtype), rand(seed + 9, (b, t, hidden), dtype))
    return p, ids, g


def rel_to_formulas(p, ids, g, got):
    """How far block_step's results are from the formulas' in 64 bits: the largest relative error in norm."""
    hidden, d = p["table"].shape[1], p["wq"].shape[0]
    P = {n: t.double().requires_grad_(n not in ("cos", "sin")) for n, t in p.items()}
    e = P["table"][ids] * math.sqrt(hidden)
    h = e + P["res"]
    y = h * (h.square().mean(-1, keepdim=True) + 1e-5).rsqrt() * P["alpha"]
    qkv = (y @ P["proj"]).view(*ids.shape, 6, d)
    c, s = P["cos"][None, :, None], P["sin"][None, :, None]

    def head(x, w):
        u = x * (x.square().mean(-1, keepdim=True) + 1e-5).rsqrt() * w
        a, b = u[..., :d // 2], u[..., d // 2:]
        return torch.cat([a * c - b * s, a * s + b * c], -1)

    oq, ok = head(qkv[..., :4, :], P["wq"]), head(qkv[..., 4:, :], P["wk"])
    loss = (oq * g[0].double()).sum() + (ok * g[1].double()).sum() + (h * g[2].double()).sum()
    loss.backward()
    want = (oq, ok, h, P["wq"].grad, P["wk"].grad, P["proj"].grad, P["alpha"].grad, P["res"].grad, P["table"].grad)
    return max(((a.double() - b).norm() / b.norm()).item() for a, b in zip(got, want))


@pytest.mark.gpu
def test_operators_together_against_64_bits(cb):
    p, ids, g = block_inputs(torch.float32, 100)
    # f32 throughout; the products (torch's, possibly with fewer bits) have 256 and 384 terms of size 1/16: in norm, errors
    # of a few hundred U of the terms, which are at most sqrt(384) times the result's size
    assert rel_to_formulas(p, ids, g, block_step(cb, p, ids, g)) <= 400 * math.sqrt(384) * U


@pytest.mark.gpu
def test_operators_together_captured_and_replayed(cb):
    """The whole step in a CUDA graph, replayed on new inputs, while an eager step runs in between."""
    p, ids, g = block_inputs(torch.bfloat16, 200)
    q, jds, h = block_inputs(torch.bfloat16, 300)
    eager = [t.clone() for t in block_step(cb, p, ids, g)]
    eager2 = [t.clone() for t in block_step(cb, q, jds, h)]
    sp, sids, sg = {n: t.clone() for n, t in p.items()}, ids.clone(), [t.clone() for t in g]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        block_step(cb, sp, sids, sg)
    torch.cuda.current_stream().wait_stream(side)
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = block_step(cb, sp, sids, sg)
    with torch.cuda.graph(other):
        outs2 = block_step(cb, q, jds, h)
    for params, i, grads, want in ((p, ids, g, eager), (q, jds, h, eager2), (p, ids, g, eager)):
        for n in sp:
            sp[n].copy_(params[n])
        sids.copy_(i)
        for a, b in zip(sg, grads):
            a.copy_(b)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other.replay()  # beside the first one
        graph.replay()
        between = block_step(cb, p, ids, g)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
        assert all(torch.equal(a, b) for a, b in zip(outs2, eager2))
        assert all(torch.equal(a, b) for a, b in zip(between, eager))


@pytest.mark.gpu
def test_operators_on_two_streams(cb):
    sets = [block_inputs(torch.bfloat16, 400 + 50 * i, b=2 + i) for i in range(2)]
    want = [[t.clone() for t in block_step(cb, *s)] for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(20):
        for i, (st, s) in enumerate(zip(streams, sets)):
            with torch.cuda.stream(st):
                got[i].append(block_step(cb, *s))
    torch.cuda.synchronize()
    for i in range(2):
        for outs in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(outs, want[i]))


@pytest.mark.gpu
def test_offsets_beyond_32_bits(cb):
    """A table and a gradient of more than 2^32 elements: the last rows are the ones whose offsets pass 32 bits."""
    if torch.cuda.get_device_properties(0).total_memory < 60 << 30:
        pytest.skip("needs 60 GB")
    hidden, vocab = 8192, (1 << 32) // 8192 + 40
    table = torch.zeros(vocab, hidden, dtype=torch.bfloat16, device="cuda")
    ids = torch.tensor([vocab - 1, 0, vocab - 1, vocab - 3], device="cuda")
    table[-1], table[-3] = 3.0, 5.0
    y = cb.embedding_scaled(table, ids, 2.0)
    assert (y[0] == 6).all() and (y[1] == 0).all() and (y[2] == 6).all() and (y[3] == 10).all()
    table.fill_(7.0)
    grad = torch.ones(4, hidden, dtype=torch.bfloat16, device="cuda")
    cb.embedding_backward(grad, ids, vocab, out=table)
    assert (table[-1] == 2).all() and (table[-3] == 1).all() and (table[0] == 1).all() and not table[-2].any() and not table[1].any()
    # the same buffer as activations of vocab rows
    x = table.fill_(1.0)
    x[-1] = 2.0
    w = torch.ones(hidden, dtype=torch.bfloat16, device="cuda")
    dx, _ = cb.rms_norm_backward(x, x, w, 0.0, out=x)
    # g == x: the gradient along x is zero up to the rounding of r, a few U of g r = 1
    assert dx[-4:].float().abs().max() <= 64 * U and dx[:4].float().abs().max() <= 64 * U
    x.fill_(1.0)
    heads = x.view(vocab * 2, 32, 128)
    k = torch.ones(vocab * 2, 1, 128, dtype=torch.bfloat16, device="cuda")
    w = torch.full((128,), 3.0, dtype=torch.bfloat16, device="cuda")
    cos, sin = torch.ones(4, 64, device="cuda"), torch.zeros(4, 64, device="cuda")
    pos = torch.ones(vocab * 2, dtype=torch.int64, device="cuda")
    cb.qk_norm_rope(heads, k, w, w, 0.0, cos, sin, positions=pos, out=(heads, k))
    assert (heads[-1] == 3).all() and (heads[0] == 3).all() and (k == 3).all()


def test_sort_digits_cover_every_key():
    """The digits of the radix sort, as the launcher cuts them: together they cover the keys 0 .. vocab."""
    for vocab in [0, 1, 2, 3, 255, 256, 511, 512, 513, 32000, 128256, 152064, (1 << 18) - 1, 1 << 18, (1 << 27) + 1, (1 << 31) - 1]:
        bits = max(1, int(vocab).bit_length())
        passes = -(-bits // 9)
        width = -(-bits // passes)
        assert width <= 9 and passes * width >= bits and (passes - 1) * width < 32
        assert np.uint32(vocab) >> np.uint32((passes - 1) * width) < (1 << width)


@pytest.mark.gpu
def test_operators_in_two_host_threads(cb):
    """Two threads on streams of their own run the step with different shapes, the first calls of the process's cached sizes
    among them."""
    import threading

    sets = [block_inputs(torch.bfloat16, 600 + 50 * i, b=2 + 3 * i, t=41 + i) for i in range(2)]
    torch.cuda.synchronize()
    got, errors = [[], []], []

    def run(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(100):
                    got[k] = [*got[k][-3:], block_step(cb, *sets[k])]
        except Exception as e:  # noqa: BLE001  (reported by the test's own thread)
            errors.append(e)

    threads = [threading.Thread(target=run, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    for k, s in enumerate(sets):
        want = block_step(cb, *s)
        for outs in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(outs, want)), k


@pytest.mark.gpu
def test_cpp_mirror_computes_what_the_package_does(cb, tmp_path):
    import os
    import shutil
    import subprocess

    gxx, cuda = shutil.which("g++"), "/usr/local/cuda"
    if gxx is None or not os.path.exists(os.path.join(cuda, "include", "cuda_runtime.h")):
        pytest.skip("no g++ or no CUDA runtime headers")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    lib_dir, exe = os.path.join(root, "candle_b200", "_lib"), str(tmp_path / "training_gpu")
    subprocess.run([gxx, "-std=c++17", "-Wall", "-Wextra", "-Werror", "-I", os.path.join(root, "include"), "-isystem", os.path.join(cuda, "include"),
                    "-o", exe, os.path.join(root, "tests", "cpp", "training_gpu.cpp"), "-L", lib_dir, "-l:libcandle_b200.so",
                    f"-Wl,-rpath,{lib_dir}", "-L", os.path.join(cuda, "lib64"), "-lcudart"], check=True)
    vocab, hidden, n, hq, hk, d, f32 = 40, 136, 90, 4, 2, 48, torch.float32
    t = {name: rand(50 + i, shape, f32) for i, (name, shape) in enumerate({
        "table": (vocab, hidden), "alpha": (hidden,), "grad": (2, n // 2, hidden), "extra": (2, n // 2, hidden), "sum": (vocab, hidden),
        "q": (n, hq, d), "k": (n, hk, d), "gq": (n, hq, d), "gk": (n, hk, d), "wq": (d,), "wk": (d,), "cos": (n, d // 2), "sin": (n, d // 2)}.items())}
    ids = make_ids(49, n, vocab, "skew").view(2, n // 2)
    for name, x in (*t.items(), ("ids", ids.to(torch.int32))):
        x.cpu().numpy().tofile(tmp_path / name)
    out = subprocess.run([exe, str(tmp_path), *map(str, (vocab, hidden, n, hq, hk, d))], capture_output=True, text=True)
    assert out.returncode == 0, (out.returncode, out.stdout + out.stderr)
    y = cb.embedding_scaled(t["table"], ids, 3.0)
    dx, dalpha = cb.rms_norm_backward(t["grad"], y, t["alpha"], 1e-5, grad_sum=t["extra"])
    heads = (t["q"], t["k"], t["wq"], t["wk"], 1e-5, t["cos"], t["sin"])
    oq, ok = cb.qk_norm_rope(*heads, interleaved=True)
    dq, dk, dwq, dwk = cb.qk_norm_rope_backward(t["gq"], t["gk"], *heads, interleaved=True)
    want = dict(y=y, dtable=cb.embedding_backward(t["grad"], ids, vocab, scale=3.0),
                sum=cb.embedding_backward(t["grad"], ids, vocab, scale=3.0, out=t["sum"].clone(), accumulate=True, padding_id=1),
                dx=dx, dalpha=dalpha, oq=oq, ok=ok, dq=dq, dk=dk, dwq=dwq, dwk=dwk)
    for name, w in want.items():
        got = torch.from_numpy(np.fromfile(tmp_path / f"out.{name}", np.float32)).view(w.shape)
        assert torch.equal(got, w.cpu()), name
