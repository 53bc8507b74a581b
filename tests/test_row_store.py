"""Feature rows held in 8 or 4 bits (psl_rows_write / psl_rows_read, point_slam_amd.row_store): refusals and the oracle's known
answers on the CPU, the kernels against the float64 oracle on the GPU.

Tolerances: none.  Scales are one fp32 division of an exact maximum, codes are correctly rounded, a value is one fp32
product rounded once more to bf16 / fp16 -- every one of these is a single IEEE operation on equal operands, so the
kernel's answer is the oracle's bit for bit."""
import ctypes as C
import os
import re
import shutil
import subprocess

import numpy as np
import pytest
import torch

from oracle import rows_oracle as RO
from point_slam_amd import _lib
from point_slam_amd.row_store import BITS, QuantizedRows
from tests.helpers import ROOT

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
gpu = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ CPU
def test_oracle_known_answers():
    x = np.zeros((1, 1, 8)); x[0, 0] = [127, 63.5, 0.5, 1.5, -0.5, -126.5, 2.4, 0]
    q, s = RO.quantize(x, "int8", 8)
    assert s[0, 0, 0] == 1.0 and list(q[0, 0]) == [127, 64, 0, 2, 0, -126, 2, 0]        # ties to even
    x[0, 0] = [448, 17, 18, 19, 2 ** -9, 2 ** -10, 3 * 2 ** -10, -464]
    q, s = RO.quantize(x * (448 / 464), "e4m3", 8)
    assert q[0, 0, 7] == -448
    assert list(RO.nearest_e4m3(np.array([17.0, 18, 19, 21, 2 ** -9, 2 ** -10, 3 * 2 ** -10]))) == \
        [16, 18, 20, 20, 2 ** -9, 0, 2 ** -8]
    x[0, 0] = [3.0, 1.5, 0, 0, 0, 0, 0, 0]
    q, s = RO.quantize(x, "int4", 8)
    # 7 * 1.5 / 3 = 3.5, but the fp32 scale 3 / 7 is a little above or below: the code follows the exact quotient
    exact = 1.5 / float(s[0, 0, 0])
    assert exact != 3.5 and q[0, 0, 1] == (4 if exact > 3.5 else 3)
    assert np.float32(1.5) / s[0, 0, 0] == np.float32(3.5)                               # what fp32 alone would see
    q, s = RO.quantize(np.array([[[np.nan, 1.0]], [[np.inf, 1.0]], [[0.0, 0.0]]]), "int8", 2)
    assert np.isnan(s[0]).all() and np.isnan(s[1]).all() and (s[2] == 0).all() and (q == 0).all()


def _args(**kw):
    buf = (C.c_char * 4096)()
    p = C.addressof(buf)
    p += -p % 16
    a = dict(format=0, dtype=0, heads=2, dim=32, group=32, rows_bits=0, n=4, capacity=8, first=0, rows=None, values=p,
             value_row_stride=64, value_head_stride=32, codes=p + 1024, codes_row_stride=64, scales=p + 2048, scales_row_stride=2, owner=None)
    a.update(kw)
    r = _lib.psl_rows_args(**a)
    r._buf = buf
    return r


@pytest.mark.parametrize("bad", [
    dict(format=3), dict(format=-1), dict(dtype=3), dict(heads=0), dict(heads=4097), dict(dim=0), dict(group=0), dict(group=24),
    dict(dim=2048, group=2048), dict(format=2, dim=33, group=11), dict(n=-1), dict(capacity=-1), dict(values=None), dict(codes=None), dict(scales=None),
    dict(first=5), dict(first=-1), dict(n=9), dict(first=2 ** 62, n=2 ** 62), dict(rows=16, rows_bits=16), dict(rows=12, rows_bits=64),
    dict(codes_row_stride=63), dict(scales_row_stride=1), dict(value_row_stride=-64)])
def test_bad_arguments_are_refused(bad):
    L = _lib.lib()
    for fn in ("psl_rows_write", "psl_rows_read"):
        rc = getattr(L, fn)(C.byref(_args(**bad)), None)
        assert rc == -1 and fn.encode() in L.psl_last_error()


def test_overlapping_output_rows_and_null_are_refused_and_nothing_is_nothing():
    L = _lib.lib()
    assert L.psl_rows_read(C.byref(_args(value_row_stride=63)), None) == -1
    assert L.psl_rows_read(C.byref(_args(value_head_stride=31)), None) == -1
    assert L.psl_rows_write(None, None) == -1 and L.psl_rows_read(None, None) == -1
    assert L.psl_rows_write(C.byref(_args(n=0, values=None)), None) == 0             # no launch: no GPU needed


def test_python_refusals():
    with pytest.raises(ValueError):
        QuantizedRows(4, fmt="int3", device="cpu")
    with pytest.raises(ValueError):
        QuantizedRows(4, dim=32, group=24, device="cpu")
    with pytest.raises(ValueError):
        QuantizedRows(4, dim=9, group=9, fmt="int4", device="cpu")
    with pytest.raises(ValueError):
        QuantizedRows(-1, device="cpu")
    st = QuantizedRows(4, device="cpu")
    v = torch.zeros(2, 2, 32)
    for bad in (v.double(), v[:, :1], v[0], torch.zeros(5, 2, 32)):
        with pytest.raises(ValueError):
            st.write(bad)
    with pytest.raises(ValueError):
        st.write(v, first=3)
    for rows in (torch.zeros(3, dtype=torch.int64), torch.zeros(2), [0, 1], torch.zeros(2, 1, dtype=torch.int64)):
        with pytest.raises(ValueError):
            st.write(v, rows=rows)
    with pytest.raises(ValueError):
        st.read(first=2, count=3)
    with pytest.raises(ValueError):
        st.read(dtype=torch.float64)
    with pytest.raises(ValueError):
        st.read(out=torch.zeros(3, 2, 32))
    with pytest.raises(_lib.PslError):
        st.write(v)                                              # no host fallback
    with pytest.raises(_lib.PslError):
        st.read()
    assert st.bytes_per_row() == 72


def test_struct_layout_matches_ctypes(tmp_path):
    if shutil.which("gcc") is None:
        pytest.skip("no gcc")
    names = [f for f, _ in _lib.psl_rows_args._fields_]
    src = tmp_path / "l.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "pointslam_hip.h"\nint main(void) {\n'
                   + "".join(f'  printf("%zu ", offsetof(psl_rows_args, {f}));\n' for f in names)
                   + '  printf("%zu", sizeof(psl_rows_args)); return 0; }\n')
    exe = tmp_path / "l"
    subprocess.check_call(["gcc", "-std=c99", "-Wall", "-pedantic", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)])
    got = [int(x) for x in subprocess.check_output([str(exe)]).split()]
    assert got == [getattr(_lib.psl_rows_args, f).offset for f in names] + [C.sizeof(_lib.psl_rows_args)]
    hdr = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "pointslam_hip.h")).read(), flags=re.S)
    body = re.search(r"typedef struct psl_rows_args \{(.*?)\} psl_rows_args;", hdr, flags=re.S).group(1)
    assert sum(st.count(",") + 1 for st in body.split(";") if st.strip()) == len(names)


# ------------------------------------------------------------------------------------------------ GPU
def _values(n, heads, dim, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    v = torch.randn(n, heads, dim, generator=g) * torch.randn(n, heads, 1, generator=g).exp() * 0.1
    # quotients on and beside the middle between two codes: the largest value over small integers
    k = torch.randint(1, 9, (n, heads, dim), generator=g).float()
    pick = torch.rand(n, heads, dim, generator=g) < 0.3
    return torch.where(pick, v.abs().amax(-1, keepdim=True) * k / 16, v).to(DT[dtype])


def _decode_codes(codes, fmt):
    """uint8 codes -> the numbers they are."""
    c = codes.cpu()
    if fmt == "int8":
        return c.view(torch.int8).double().numpy()
    if fmt == "e4m3":
        return c.view(torch.float8_e4m3fn).double().numpy()
    q = torch.stack([c & 15, c >> 4], -1).flatten(-2).to(torch.int8)
    return torch.where(q > 7, q - 16, q).double().numpy()


def _same(a, b):
    return np.array_equal(np.asarray(a), np.asarray(b), equal_nan=True)


def _expect(v, fmt, group, dtype):
    q, s = RO.quantize(v.float().cpu().numpy(), fmt, group)
    return q, s, torch.from_numpy(RO.values(q, s)).to(dtype)


@gpu
@pytest.mark.parametrize("fmt", ["int8", "e4m3", "int4"])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("group", [1022, 1020, 1016, 1021])
def test_a_read_is_the_fp32_value_converted(fmt, dtype, group):
    """In pieces of two, four, eight and one: about one product in 2^14 lies, once it is an fp32 number, in the middle between two
    fp16 ones, and is then rounded again; rounding the exact product would give the other one for half of them."""
    if fmt == "int4" and group % 2:
        group = 1010
    st = QuantizedRows(1000, 1, group, fmt, group).write(torch.randn(1000, 1, group, generator=torch.Generator().manual_seed(3)).cuda())
    assert torch.equal(st.read(dtype=DT[dtype]), st.read().to(DT[dtype]))


@gpu
@pytest.mark.parametrize("fmt", ["int8", "e4m3", "int4"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,heads,dim,group", [(1, 1, 2, 2), (3, 2, 32, 32), (257, 2, 32, 8), (65, 3, 80, 80), (129, 8, 128, 32),
                                               (17, 1, 1024, 1024), (5, 5, 66, 22), (33, 1, 36, 12), (2, 1, 4096, 256), (9, 2, 514, 514),
                                               (70, 4, 200, 40)])
def test_write_and_read_match_the_oracle(fmt, dtype, n, heads, dim, group):
    v = _values(n, heads, dim, dtype, seed=n + dim)
    st = QuantizedRows(n + 2, heads, dim, fmt, group)
    st.write(v.cuda(), first=1)
    q, s, want = _expect(v, fmt, group, DT[dtype])
    assert _same(st.scales[1:n + 1].cpu().numpy(), s)
    assert _same(_decode_codes(st.codes[1:n + 1], fmt), q)
    assert _same(st.read(first=1, count=n, dtype=DT[dtype]).float().cpu(), want.float())
    assert (st.codes[0] == 0).all() and (st.codes[n + 1] == 0).all() and (st.scales[[0, n + 1]] == 0).all()
    full = st.read()
    assert full.dtype == torch.float32 and _same(full[1:n + 1].cpu(), RO.values(q, s)) and (full[0] == 0).all()


@gpu
@pytest.mark.parametrize("fmt,dim,group", [("int8", 1, 1), ("e4m3", 33, 11), ("int8", 1021, 1021), ("e4m3", 77, 7)])
def test_odd_groups(fmt, dim, group):
    v = _values(19, 3, dim, "f32")
    st = QuantizedRows(19, 3, dim, fmt, group).write(v.cuda())
    q, s, want = _expect(v, fmt, group, torch.float32)
    assert _same(st.scales.cpu(), s) and _same(_decode_codes(st.codes, fmt), q) and _same(st.read().cpu(), want)


@gpu
@pytest.mark.parametrize("fmt", ["int8", "e4m3", "int4"])
def test_every_quotient_of_a_dense_sweep_is_rounded_right(fmt):
    """All 2^16 bf16 patterns as values beside a few maxima: ties, subnormal codes, signs, zeros of either sign."""
    bits = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(torch.bfloat16).float()
    bits = bits[torch.isfinite(bits)]
    rows = []
    for top in (1.0, 3.0, 0.7421875, 447.0, 1e-30, 3.0e38, 2.0 ** -126, 1e-42):
        x = bits[bits.abs() <= top]
        pad = -x.numel() % 31
        x = torch.cat([x, torch.zeros(pad)]).reshape(-1, 31)
        rows.append(torch.cat([x, torch.full((x.shape[0], 1), top)], 1))
    v = torch.cat(rows)[:, None, :]
    st = QuantizedRows(v.shape[0], 1, 32, fmt).write(v.cuda())
    q, s, want = _expect(v, fmt, 32, torch.float32)
    assert _same(st.scales.cpu(), s)
    got = _decode_codes(st.codes, fmt)
    bad = np.flatnonzero((got != q).any(-1).ravel())
    assert bad.size == 0, (bad[:5], v[bad[:1]], got[bad[:1]], q[bad[:1]])
    assert _same(st.read().cpu(), want)


@gpu
def test_zeros_infinities_and_nan():
    v = torch.randn(6, 2, 32)
    v[0] = 0; v[1, 0, 3] = float("inf"); v[2, 1, 31] = float("nan"); v[3, 0, 0] = -float("inf"); v[4] = 1.4e-45; v[5, 0] = -0.0
    for fmt in ("int8", "e4m3", "int4"):
        st = QuantizedRows(6, 2, 32, fmt).write(v.cuda())
        out = st.read().cpu()
        q, s, want = _expect(v, fmt, 32, torch.float32)
        assert _same(out, want)
        assert (out[0] == 0).all() and out[1, 0].isnan().all() and out[2, 1].isnan().all() and out[3, 0].isnan().all()
        assert not out[1, 1].isnan().any() and not out[2, 0].isnan().any() and (out[4] == 0).all()


@gpu
@pytest.mark.parametrize("ids", [torch.int32, torch.int64])
def test_scattered_rows_padding_and_rows_left_alone(ids):
    v = _values(64, 2, 32, "f32")
    st = QuantizedRows(200, 2, 32, "int8")
    before = _values(200, 2, 32, "f32", seed=5)
    st.write(before.cuda())
    base = st.read().cpu()
    rows = torch.randperm(200, generator=torch.Generator().manual_seed(1))[:64].to(ids)
    rows[::7] = -1
    rows[3], rows[5] = 200, torch.iinfo(ids).max
    rows[6] = torch.iinfo(ids).min
    st.write(v.cuda(), rows=rows.cuda(), distinct=True)
    _, _, want = _expect(v, "int8", 32, torch.float32)
    expect = base.clone()
    ok = (rows >= 0) & (rows < 200)
    expect[rows[ok].long()] = want[ok]
    assert _same(st.read().cpu(), expect)
    got = st.read(rows=rows.cuda()).cpu()
    assert _same(got[ok], want[ok]) and (got[~ok] == 0).all()
    twice = st.read(rows=torch.tensor([3, 3, 199, 3]).cuda()).cpu()
    assert _same(twice, expect[[3, 3, 199, 3]])


@gpu
@pytest.mark.parametrize("ids", [torch.int32, torch.int64])
def test_the_last_of_several_writes_to_a_row_wins(ids):
    n = 5000
    v = _values(n, 2, 32, "bf16")
    rows = torch.randint(-2, 40, (n,), generator=torch.Generator().manual_seed(2))
    _, _, want = _expect(v, "e4m3", 32, torch.float32)
    last = {}
    for i, r in enumerate(rows.tolist()):
        last[r] = i
    for rep in range(5):
        st = QuantizedRows(38, 2, 32, "e4m3")          # ids 38, 39 fall outside
        st.write(v.cuda(), rows=rows.to(ids).cuda())
        out = st.read().cpu()
        for r in range(38):
            assert _same(out[r], want[last[r]]), (rep, r)


@gpu
@pytest.mark.parametrize("fmt", ["int8", "e4m3", "int4"])
@pytest.mark.parametrize("off", [0, 1, 2, 3])
def test_strided_and_misaligned_values(fmt, off):
    """Values inside wider records, off the 16-byte grid; heads in another order; a broadcast row; a strided output."""
    rec = _values(50, 1, 80, "f32").reshape(50, 80)
    v = torch.as_strided(rec, (50, 2, 32), (80, 40, 1), off)
    st = QuantizedRows(50, 2, 32, fmt).write(torch.as_strided(rec.cuda(), (50, 2, 32), (80, 40, 1), off))
    _, _, want = _expect(v, fmt, 32, torch.float32)
    assert _same(st.read().cpu(), want)
    out = torch.full((50, 90), 7.0, device="cuda")
    view = torch.as_strided(out, (50, 2, 32), (90, 41, 1), off)
    st.read(out=view)
    assert _same(view.cpu(), want)
    mask = torch.ones(50, 90, dtype=torch.bool)
    torch.as_strided(mask, (50, 2, 32), (90, 41, 1), off).fill_(False)
    assert (out.cpu()[mask] == 7.0).all()
    h = torch.randn(2, 50, 32)
    assert _same(QuantizedRows(50, 2, 32, fmt).write(h.cuda().transpose(0, 1)).read().cpu(), _expect(h.transpose(0, 1), fmt, 32, torch.float32)[2])
    one = torch.randn(1, 2, 32)
    assert _same(QuantizedRows(50, 2, 32, fmt).write(one.cuda().expand(50, 2, 32)).read().cpu(), _expect(one.expand(50, 2, 32), fmt, 32, torch.float32)[2])
    t = torch.randn(50, 32, 2)
    assert _same(QuantizedRows(50, 2, 32, fmt).write(t.cuda().transpose(1, 2)).read().cpu(), _expect(t.transpose(1, 2), fmt, 32, torch.float32)[2])
    half = _values(50, 1, 81, "bf16").reshape(50, 81)
    hv = torch.as_strided(half, (50, 2, 32), (81, 40, 1), off)
    assert _same(QuantizedRows(50, 2, 32, fmt).write(torch.as_strided(half.cuda(), (50, 2, 32), (81, 40, 1), off)).read().cpu(), _expect(hv, fmt, 32, torch.float32)[2])


@gpu
def test_nothing_to_do():
    st = QuantizedRows(0)
    assert st.read().shape == (0, 2, 32)
    assert (st.read(rows=torch.tensor([0, -1], device="cuda")) == 0).all()
    st.write(torch.zeros(2, 2, 32, device="cuda"), rows=torch.tensor([0, 5], device="cuda"))
    st = QuantizedRows(3)
    st.write(torch.zeros(0, 2, 32, device="cuda"))
    st.write(torch.zeros(0, 2, 32, device="cuda"), rows=torch.zeros(0, dtype=torch.int64, device="cuda"))
    assert st.read(count=0).shape == (0, 2, 32) and (st.read() == 0).all()


@gpu
def test_another_stream_and_a_captured_graph():
    v = _values(300, 2, 32, "f32").cuda()
    rows = torch.randperm(400)[:300].cuda()
    want = QuantizedRows(400).write(v, rows=rows).read(rows=rows)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = QuantizedRows(400).write(v, rows=rows).read(rows=rows)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    st, inp, ids, out = QuantizedRows(400), v.clone(), rows.clone(), torch.empty_like(v)
    st.write(inp, rows=ids).read(rows=ids, out=out)          # warm-up
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        st.write(inp, rows=ids)
        st.read(rows=ids, out=out)
    for k in range(4):
        inp.copy_(v * (k + 1)); ids.copy_((rows + k) % 400)
        if k == 2:
            ids[:100] = ids[100:200]                          # the same id twice, the later one holds
        g.replay()
        eager = QuantizedRows(400).write(inp, rows=ids).read(rows=ids)
        torch.cuda.synchronize()
        assert torch.equal(out, eager), k


@gpu
def test_offsets_past_32_bits_and_more_rows_than_one_launch_takes():
    st = QuantizedRows(4_400_000, 8, 128, "int8")             # 4.5 GB of codes
    rows = torch.tensor([0, 2 ** 21 - 1, 2 ** 21, 2 ** 22 - 1, 2 ** 22, 4_399_999])
    v = _values(6, 8, 128, "bf16")
    st.write(v.cuda(), rows=rows.cuda())
    want = _expect(v, "int8", 128, torch.bfloat16)[2]
    assert _same(st.read(rows=rows.cuda(), dtype=torch.bfloat16).float().cpu(), want.float())
    assert (st.scales.sum(-1).sum(-1) != 0).sum() == 6
    del st
    n = (1 << 20) + 40                                        # 2^30 threads end after 2^20 rows of 1024 groups
    x = torch.randn(64, 1, 1024).to(torch.float16)
    big = x.cuda().repeat(n // 64 + 1, 1, 1)[:n]
    st = QuantizedRows(n, 1, 1024, "int8", 1).write(big)
    out = st.read(dtype=torch.float16)
    want = _expect(x, "int8", 1, torch.float16)[2].cuda()
    for lo in (0, (1 << 20) - 64, (1 << 20) - 32, n - 64):
        assert torch.equal(out[lo:lo + 64], want[(torch.arange(lo, lo + 64) % 64).cuda()]), lo


@gpu
def test_tensors_of_another_device():
    if torch.cuda.device_count() < 2:
        pytest.skip("one GPU")
    v = torch.randn(10, 2, 32)
    st = QuantizedRows(10, device="cuda:1").write(v.to("cuda:1"))
    assert _same(st.read().cpu(), _expect(v, "int8", 32, torch.float32)[2])
    with pytest.raises(ValueError):
        st.write(v.to("cuda:0"))


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("fmt", ["int8", "e4m3", "int4"])
def test_groups_of_the_smallest_numbers(fmt, dtype):
    """Groups whose largest value is 0 to 600 times the smallest denormal: where the scale underflows to 0 every code is 0, and what is
    read is 0 and not -0 in the integer formats; from there on codes are nearest to the quotient by a scale of few bits."""
    tops = torch.arange(0, 601, dtype=torch.int32)
    bits = tops[:, None] * torch.tensor([4, 3, 2, 1], dtype=torch.int32) // 4
    v = (bits.view(torch.float32) if dtype == "f32" else bits.to(torch.int16).view(torch.bfloat16))
    v = (v * torch.tensor([1, -1, 1, -1], dtype=v.dtype))[:, None, :]
    assert int((v.float().abs().amax(-1) > 0).sum()) == 600
    st = QuantizedRows(601, 1, 4, fmt).write(v.cuda())
    q, s, want = _expect(v, fmt, 4, DT[dtype])
    assert _same(st.scales.cpu(), s) and (dtype == "bf16" or (s[1:4] == 0).all())
    assert _same(_decode_codes(st.codes, fmt), q)
    out = st.read(dtype=DT[dtype]).cpu()
    assert _same(out.float(), want.float())
    if fmt != "e4m3":
        assert (st.codes.cpu()[torch.from_numpy(s[..., 0] == 0)] == 0).all()
        assert not torch.signbit(out[out == 0]).any()


@gpu
@pytest.mark.parametrize("fmt", ["int8", "e4m3", "int4"])
def test_groups_of_the_largest_numbers_read_back_finite(fmt):
    """Up to fp32's largest number, of either sign (what a mask of the type's lowest value is): no finite group reads back as an
    infinity, and every value is as near as elsewhere."""
    top = torch.full((40,), torch.finfo(torch.float32).max).view(torch.int32) - torch.arange(40, dtype=torch.int32)
    v = torch.zeros(40, 1, 8)
    v[:, 0, 0] = top.view(torch.float32)
    v[:, 0, 1], v[:, 0, 2], v[:, 0, 3] = -v[:, 0, 0], v[:, 0, 0] / 2, -v[:, 0, 0] / 3
    v[::2, 0, 0] = 0.0                                        # the negative one by itself
    st = QuantizedRows(40, 1, 8, fmt).write(v.cuda())
    q, s, want = _expect(v, fmt, 8, torch.float32)
    out = st.read().cpu()
    assert torch.isfinite(out).all() and _same(st.scales.cpu(), s) and _same(_decode_codes(st.codes, fmt), q) and _same(out, want)
    # half a code step: of the scale for integers, 2^-4 of the value for e4m3; and the product's rounding
    step = torch.from_numpy(s).double() / 2 if fmt != "e4m3" else v.double().abs() * 2.0 ** -4
    assert ((out.double() - v.double()).abs() <= step + v.double().abs() * 2.0 ** -23).all()


@gpu
@pytest.mark.parametrize("fmt", ["int8", "int4"])
def test_a_read_into_heads_that_follow_one_another(fmt):
    """[heads, n, dim] memory seen as [n, heads, dim]: a row of one head lies between the heads of another, and none overlap."""
    v = _values(37, 3, 32, "f32")
    st = QuantizedRows(37, 3, 32, fmt).write(v.cuda())
    _, _, want = _expect(v, fmt, 32, torch.float32)
    for pad in (0, 8):
        out = torch.full((3, 37, 32 + pad), 7.0, device="cuda")
        st.read(out=out[:, :, :32].transpose(0, 1))
        assert _same(out[:, :, :32].transpose(0, 1).cpu(), want) and (out[:, :, 32:] == 7.0).all()
        rows = torch.tensor([5, -1, 36, 5], device="cuda")
        few = torch.full((3, 4, 32 + pad), 7.0, device="cuda")
        st.read(rows=rows, out=few[:, :, :32].transpose(0, 1))
        expect = want[[5, 0, 36, 5]]
        expect[1] = 0
        assert _same(few[:, :, :32].transpose(0, 1).cpu(), expect)


def test_outputs_whose_rows_overlap_are_refused_in_either_order():
    L = _lib.lib()
    for kw in (dict(value_row_stride=32, value_head_stride=127), dict(value_row_stride=31, value_head_stride=128), dict(value_row_stride=0, value_head_stride=128),
               dict(value_row_stride=40, value_head_stride=40), dict(value_row_stride=64, value_head_stride=0), dict(value_row_stride=33, value_head_stride=32)):
        assert L.psl_rows_read(C.byref(_args(**kw)), None) == -1 and b"overlap" in L.psl_last_error(), kw
