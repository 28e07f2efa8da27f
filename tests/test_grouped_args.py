"""CPU tests of the argument checks of the scaled 8-bit and the expert-grouped products: every refusal is a status and a
message before anything touches CUDA. Addresses are made up and never dereferenced."""
import os
import random
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

from tiledcuda_b200 import _lib, ops

F32, F16, I32, BF16 = 0, 1, 2, 4
BAD, UNSUPPORTED = -1, -2


def quantize(l, x=64, q=64, s=64, rows=4, cols=8, ldx=8, ldq=8, ty=F16):
    return l.tc_quantize_rows(x, q, s, rows, cols, ldx, ldq, ty, None)


def i8(l, a=64, b=64, sa=64, sb=64, c=4096, m=4, n=8, k=32, lda=32, ldb=32, ldc=8, ty=F16):
    return l.tc_gemm_i8(a, b, sa, sb, c, m, n, k, lda, ldb, ldc, ty, None)


def grouped(l, a=64, b=64, off=64, wide=0, c=4096, rows=4, e=2, n=8, k=32, lda=32, ldb=32, sb=256, ldc=8, it=F16, ct=F16):
    return l.tc_grouped_gemm(a, b, off, wide, c, rows, e, n, k, lda, ldb, sb, ldc, it, ct, None)


def grouped_i8(l, a=64, b=64, sa=64, sb=64, off=64, wide=0, c=4096, rows=4, e=2, n=8, k=32, lda=32, ldb=32, stride=256, ldc=8, ct=F16):
    return l.tc_grouped_gemm_i8(a, b, sa, sb, off, wide, c, rows, e, n, k, lda, ldb, stride, ldc, ct, None)


def dgrad(l, dc=64, b=64, off=64, wide=0, da=4096, rows=4, e=2, n=8, k=32, lddc=8, ldb=32, sb=256, ldda=32, it=F16, ot=F16):
    return l.tc_grouped_gemm_dgrad(dc, b, off, wide, da, rows, e, n, k, lddc, ldb, sb, ldda, it, ot, None)


def wgrad(l, dc=64, a=64, off=64, wide=0, db=4096, rows=4, e=2, n=8, k=32, lddc=8, lda=32, lddb=32, sdb=256, it=F16, ot=F16):
    return l.tc_grouped_gemm_wgrad(dc, a, off, wide, db, rows, e, n, k, lddc, lda, lddb, sdb, it, ot, None)


CASES = [
    (quantize, dict(x=None), BAD, "null"), (quantize, dict(s=None), BAD, "null"), (quantize, dict(cols=0), BAD, "positive"),
    (quantize, dict(rows=-1), BAD, "negative"), (quantize, dict(rows=1 << 31), BAD, "31 bits"), (quantize, dict(ldx=7), BAD, "leading dimension"),
    (quantize, dict(ldq=7), BAD, "leading dimension"), (quantize, dict(ty=I32), BAD, "x_type"), (quantize, dict(x=65), BAD, "aligned"),
    (quantize, dict(q=128), BAD, "overlap"), (quantize, dict(s=128), BAD, "overlap"), (quantize, dict(x=128), BAD, "overlap"),
    (i8, dict(a=None), BAD, "null"), (i8, dict(sa=None), BAD, "null"), (i8, dict(c=None), BAD, "null"), (i8, dict(m=-1), BAD, "negative"),
    (i8, dict(n=0), BAD, "positive"), (i8, dict(k=0), BAD, "positive"), (i8, dict(lda=40), BAD, "row stride"), (i8, dict(ldb=24), BAD, "leading dimension"),
    (i8, dict(ldc=7), BAD, "leading dimension"), (i8, dict(a=72), BAD, "aligned"), (i8, dict(c=65), BAD, "aligned"), (i8, dict(sb=66), BAD, "aligned"),
    (i8, dict(ty=I32), BAD, "c_type"), (i8, dict(k=131072, lda=131072, ldb=131072), UNSUPPORTED, "overflow"), (i8, dict(n=1 << 31), BAD, "31 bits"),
    (i8, dict(lda=1 << 40), BAD, "too large"),
    (grouped, dict(off=None), BAD, "offsets"), (grouped, dict(off=66), BAD, "aligned"), (grouped, dict(off=68, wide=1), BAD, "aligned"),
    (grouped, dict(e=0), BAD, "positive"), (grouped, dict(e=1025), UNSUPPORTED, "1024"), (grouped, dict(rows=-1), BAD, "negative"),
    (grouped, dict(lda=36), BAD, "row stride"), (grouped, dict(ldb=36), BAD, "row stride"), (grouped, dict(sb=260), BAD, "expert stride"),
    (grouped, dict(sb=16), BAD, "expert stride"), (grouped, dict(sb=0), BAD, "expert stride"), (grouped, dict(it=F32, ct=F32), BAD, "in_type"), (grouped, dict(ct=BF16), BAD, "input's type"),
    (grouped, dict(b=72), BAD, "aligned"), (grouped, dict(ldc=0), BAD, "leading dimension"), (grouped, dict(sb=1 << 40), BAD, "too large"),
    (grouped, dict(c=64), BAD, "overlap"), (grouped, dict(rows=(1 << 31) - 1), BAD, "31 bits"),
    (grouped, dict(k=1 << 28, lda=1 << 28, ldb=1 << 28, sb=1 << 31), UNSUPPORTED, "terms"), (i8, dict(c=64), BAD, "overlap"),
    (dgrad, dict(da=64), BAD, "overlap"), (dgrad, dict(n=1 << 28, lddc=1 << 28), UNSUPPORTED, "terms"),
    (wgrad, dict(db=64), BAD, "overlap"), (wgrad, dict(rows=1 << 28), UNSUPPORTED, "terms"),
    (grouped_i8, dict(off=None), BAD, "offsets"), (grouped_i8, dict(stride=264), BAD, "expert stride"), (grouped_i8, dict(lda=40), BAD, "row stride"),
    (grouped_i8, dict(k=1 << 18, lda=1 << 18, ldb=1 << 18, stride=1 << 21), UNSUPPORTED, "overflow"), (grouped_i8, dict(sa=None), BAD, "null"),
    (dgrad, dict(lddc=12), BAD, "row stride"), (dgrad, dict(ldda=31), BAD, "leading dimension"), (dgrad, dict(dc=None), BAD, "null"),
    (dgrad, dict(ot=BF16), BAD, "input's type"), (dgrad, dict(e=1025), UNSUPPORTED, "1024"), (dgrad, dict(off=None), BAD, "offsets"),
    (wgrad, dict(lddc=12), BAD, "row stride"), (wgrad, dict(lda=36), BAD, "row stride"), (wgrad, dict(db=None), BAD, "null"), (wgrad, dict(db=None, rows=0), BAD, "null"),
    (wgrad, dict(lddb=31), BAD, "leading dimension"), (wgrad, dict(sdb=8), BAD, "expert stride"), (wgrad, dict(it=I32, ot=I32), BAD, "in_type"),
    (wgrad, dict(off=None), BAD, "offsets"),
]


@pytest.mark.parametrize("call,change,status,needle", CASES)
def test_refusals(call, change, status, needle):
    lib = _lib.load()
    assert call(lib, **change) == status
    assert needle in lib.tc_last_error().decode()


def test_no_rows_is_no_work():
    lib = _lib.load()
    assert quantize(lib, x=None, q=None, s=None, rows=0) == 0
    assert i8(lib, a=None, c=None, sa=None, m=0) == 0
    assert grouped(lib, a=None, c=None, rows=0) == 0
    assert grouped_i8(lib, a=None, c=None, sa=None, rows=0) == 0
    assert dgrad(lib, dc=None, da=None, rows=0) == 0


def test_python_route_refuses_cpu_tensors_and_wrong_types():
    a, b, c = torch.zeros(4, 16, dtype=torch.float16), torch.zeros(2, 8, 16, dtype=torch.float16), torch.zeros(4, 8, dtype=torch.float16)
    off = torch.tensor([0, 2, 4], dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.grouped_gemm(a, b, off, c)
    with pytest.raises(ValueError, match="CUDA"):
        ops.grouped_gemm_dgrad(c, b, off, a)
    with pytest.raises(ValueError, match="CUDA"):
        ops.grouped_gemm_wgrad(c, a, off, b)
    with pytest.raises(ValueError, match="CUDA"):
        ops.quantize_rows(a, a.to(torch.int8), torch.zeros(4))
    with pytest.raises(ValueError, match="CUDA"):
        ops.gemm_i8(a.to(torch.int8), b[0].to(torch.int8), torch.zeros(4), torch.zeros(8), c)
    with pytest.raises(ValueError, match="3-D"):
        ops.grouped_gemm(a, b[0], off, c)
    with pytest.raises(TypeError):
        ops.grouped_gemm(None, b, off, c)
    with pytest.raises(TypeError):
        ops.quantize_rows([1.0], None, None)


@pytest.mark.parametrize("file", [None, b"not a library"])
def test_an_op_library_that_does_not_load_leaves_the_other_route(tmp_path, monkeypatch, file):
    path = tmp_path / "libtiledcuda.so"
    if file is not None:
        path.write_bytes(file)
    monkeypatch.setattr(ops, "_OP_LIB", path)
    monkeypatch.setattr(ops, "_registered_ops", None)
    assert all(ops._registered(name) is None for name in ("gemm_i8", "grouped_gemm_wgrad"))


def test_direct_calls_leave_what_is_not_for_them():
    calls = pytest.importorskip("tiledcuda_b200._calls")
    t = [torch.zeros(4, 16, dtype=torch.int8), torch.zeros(8, 16, dtype=torch.int8), torch.zeros(4), torch.zeros(8), torch.zeros(4, 8)]
    assert calls.gemm_i8(*t) is False
    assert calls.gemm_i8(*t[:4]) is False
    assert calls.gemm_i8(None, *t[1:]) is False
    assert calls.gemm_i8() is False


@pytest.fixture()
def shapes_on_a_gpu(monkeypatch):
    """CUDA tensors without a GPU, for the way a call takes; whatever is launched in the end is an error."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    def launched(*args):
        raise AssertionError("launched")

    monkeypatch.setattr(ops, "_launch", launched)
    monkeypatch.setattr(ops, "_registered_ops", {})
    monkeypatch.setattr(ops, "_direct_calls", {})
    with FakeTensorMode(allow_non_fake_inputs=True):
        yield [torch.empty(4, 16, dtype=torch.int8, device="cuda"), torch.empty(8, 16, dtype=torch.int8, device="cuda"),
               torch.empty(4, device="cuda"), torch.empty(8, device="cuda"), torch.empty(4, 8, device="cuda")]


@pytest.mark.parametrize("error", [RuntimeError("not here"), TypeError("nor there"), NotImplementedError("no such kernel")])
def test_an_error_of_the_op_is_raised_and_nothing_else_launched(shapes_on_a_gpu, error):
    calls = []

    def op(*args):
        calls.append(args)
        raise error

    ops._registered_ops["gemm_i8"] = op
    with pytest.raises(type(error), match=str(error)):
        ops.gemm_i8(*shapes_on_a_gpu)
    assert len(calls) == 1
    with pytest.raises(ValueError, match="scale_a must be"):   # what the checks can explain they do
        ops.gemm_i8(*shapes_on_a_gpu[:2], shapes_on_a_gpu[3], *shapes_on_a_gpu[3:])


def test_what_the_c_entry_point_refused_is_raised_as_such(shapes_on_a_gpu):
    calls = []

    def op(*args):
        calls.append(args)
        raise RuntimeError("tiledcuda::gemm_i8 failed with status -3: a call failed\nbacktrace")

    ops._registered_ops["gemm_i8"] = op
    with pytest.raises(_lib.TiledCudaError, match="tc_gemm_i8 failed with status -3: a call failed$") as raised:
        ops.gemm_i8(*shapes_on_a_gpu)
    assert raised.value.status == -3 and len(calls) == 1
    ops._registered_ops["gemm_i8"] = lambda *args: calls.append(args)
    ops._direct_calls["gemm_i8"] = op   # past the dispatcher: not made again through it
    with pytest.raises(_lib.TiledCudaError, match="a call failed"):
        ops.gemm_i8(*shapes_on_a_gpu)
    assert len(calls) == 2


def test_without_the_op_the_c_entry_point_is_called(shapes_on_a_gpu, monkeypatch):
    names = []
    monkeypatch.setattr(ops, "_launch", lambda name, *args: names.append(name))
    monkeypatch.setattr(torch.Tensor, "data_ptr", lambda t: 64)
    ops.gemm_i8(*shapes_on_a_gpu)
    assert names == ["tc_gemm_i8"]


# An operand as (address, bytes of a row, rows, bytes from row to row, slices, bytes from slice to slice), byte by byte.
def covered(base, width, rows=1, step=0, slices=1, slice_step=0):
    count = np.zeros(1 << 15, dtype=np.int32)
    for e in range(slices):
        for r in range(rows):
            at = base + e * slice_step + r * step
            count[at:at + width] += 1
    return count


def random_overlap_calls(rng):
    """(call, whether the output meets an operand or itself): layouts in a few kilobytes, dense, with gaps and interleaved."""
    def addr(granule, top=4096):
        return rng.randrange(0, top, granule)

    def stack(e, n, k, granule, shared=False):
        """row and expert stride"""
        k = -(-k // granule) * granule
        ld = k + rng.choice([0, 0, 0, granule, 3 * granule, 10 * granule])
        return rng.choice([(ld, n * ld), (ld, n * ld + 2 * granule), (e * ld, ld), (e * ld + 5 * granule, ld)] + [(ld, max(k, ld * n // 2 // granule * granule))] * shared)

    kind = rng.choice(["quantize", "i8", "grouped", "dgrad", "wgrad"])
    m, n, k, e = rng.randrange(1, 7), rng.randrange(1, 12), rng.randrange(1, 12), rng.randrange(1, 4)
    if kind == "quantize":
        x, q, s, ldx, ldq = addr(2), addr(1), addr(4), k + rng.choice([0, 0, 1, 7, 20]), k + rng.choice([0, 0, 2, 13, k + 20])
        if rng.random() < 0.3:
            ldq = 2 * ldx
        parts = [covered(x, 2 * k, m, 2 * ldx), covered(q, k, m, ldq), covered(s, 4 * m)]
        return (lambda l, b: l.tc_quantize_rows(b + x, b + q, b + s, m, k, ldx, ldq, F16, None)), (sum(p > 0 for p in parts) > 1).any()
    a, b, off, sa, sb, c = addr(16), addr(16), addr(8), addr(4), addr(4), addr(4)
    esz, ct = rng.choice([(4, F32), (2, F16)])
    if kind == "i8":
        lda, ldb, ldc = (16 * rng.randrange(1, 6) for _ in range(3))
        ins = [covered(a, k, m, lda), covered(b, k, n, ldb), covered(sa, 4 * m), covered(sb, 4 * n)]
        out = covered(c, n * esz, m, ldc * esz)
        return (lambda l, p: l.tc_gemm_i8(p + a, p + b, p + sa, p + sb, p + c, m, n, k, lda, ldb, ldc, ct, None)), (sum(i > 0 for i in ins) * out > 0).any()
    ld_in = -(-max(n, k) // 8) * 8 + rng.choice([0, 8, 40])
    if kind == "wgrad":
        ld, stride = stack(e, n, k, 1, True)
        ins = [covered(a, 2 * n, m, 2 * ld_in), covered(b, 2 * k, m, 2 * ld_in), covered(off, 4 * (e + 1))]
        out = covered(c, k * esz, n, ld * esz, e, stride * esz)
        return (lambda l, p: l.tc_grouped_gemm_wgrad(p + a, p + b, p + off, 0, p + c, m, e, n, k, ld_in, ld_in, ld, stride, F16, ct, None),
                (out > 1).any() or (sum(i > 0 for i in ins) * out > 0).any())
    ld, stride = stack(e, n, k, 8, True)
    wide = rng.randrange(2)
    ins = [covered(b, 2 * k, n, 2 * ld, e, 2 * stride), covered(off, (8 if wide else 4) * (e + 1))]
    ldo = rng.choice([12, 24, ld_in, 2 * ld_in, 100])
    if kind == "grouped":
        ins.append(covered(a, 2 * k, m, 2 * ld_in))
        out = covered(c, n * esz, m, ldo * esz)
        call = lambda l, p: l.tc_grouped_gemm(p + a, p + b, p + off, wide, p + c, m, e, n, k, ld_in, ld, stride, ldo, F16, ct, None)
    else:
        ins.append(covered(a, 2 * n, m, 2 * ld_in))
        out = covered(c, k * esz, m, ldo * esz)
        call = lambda l, p: l.tc_grouped_gemm_dgrad(p + a, p + b, p + off, wide, p + c, m, e, n, k, ld_in, ld, stride, ldo, F16, ct, None)
    return call, (sum(i > 0 for i in ins) * out > 0).any()


def check_random_overlaps():
    """In a process that sees no GPU: a call that passes the checks ends with the failure to find one."""
    lib, rng, seen = _lib.load(), random.Random(0), [0, 0]
    for _ in range(4000):
        call, meets = random_overlap_calls(rng)
        status = call(lib, 1 << 20)
        text = lib.tc_last_error().decode()
        assert (status, "overlap" in text) == ((BAD, True) if meets else (-3, False)), (status, text, meets)
        seen[int(meets)] += 1
    assert min(seen) > 500, seen


def test_outputs_that_overlap_an_operand_are_refused_and_others_are_not():
    code = "import sys; sys.path[:0] = sys.argv[1:]; import test_grouped_args as t; t.check_random_overlaps()"
    here = Path(__file__).resolve().parent
    done = subprocess.run([sys.executable, "-c", code, str(here), str(here.parent)], env={**os.environ, "CUDA_VISIBLE_DEVICES": ""}, capture_output=True, text=True)
    assert done.returncode == 0, done.stderr[-2000:]


@pytest.mark.parametrize("call,change", [
    (quantize, dict(x=4096, q=4096 + 63, s=64)), (quantize, dict(x=4096, q=8192, s=4096 + 60)), (quantize, dict(x=4096, q=8192, s=8192 + 28)),
    (i8, dict(c=64 + 96)), (i8, dict(a=4096, c=4048)), (i8, dict(sa=4096 + 60)), (i8, dict(sb=4096 + 4)),
    (grouped, dict(a=4096 + 16)), (grouped, dict(b=4096 - 1024 + 16)), (grouped, dict(off=4096 + 60)), (grouped, dict(off=4096 - 16, wide=1)),
    (grouped_i8, dict(sb=4096 - 60)), (grouped_i8, dict(c=64 + 480)), (dgrad, dict(b=4096 + 240)), (dgrad, dict(dc=4096 - 48)),
    (wgrad, dict(a=4096 + 1008)), (wgrad, dict(dc=4096 - 16)), (wgrad, dict(off=4096, rows=0)), (wgrad, dict(sdb=32)), (wgrad, dict(lddb=64)),
])
def test_partial_overlaps_are_refused(call, change):
    lib = _lib.load()
    assert call(lib, **change) == BAD
    assert "overlap" in lib.tc_last_error().decode()
