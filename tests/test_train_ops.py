"""The training-step operators (sum with dropout, balance loss, policy loss):
refusals and layouts on the CPU, numerics on the GPU against 64-bit numpy
(oracle/train_ref.py). Every bound below is counted from the operations a
value goes through, u = 2^-24 for each in fp32, and half a step of the output's
type for its one rounding."""
import os
import subprocess

import numpy as np
import pytest

import xucg_amd
from oracle import train_ref as R
from xucg_amd import _lib
from xucg_amd import group as G

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
U = 2.0 ** -24
DTS = ["float32", "bfloat16", "float16"]
DT = {name: i for i, name in enumerate(_lib.DTYPES)}
INVALID, UNSUPPORTED = _lib.UCS_ERR_INVALID_PARAM, _lib.UCS_ERR_UNSUPPORTED
PTR = 1 << 20         # an address that a refused call never looks at


# ---- CPU ---------------------------------------------------------------------------
def test_philox_known_answers():
    """The published known-answer vectors of Philox-4x32-10."""
    f = 0xffffffff
    for ctr, key, want in (
            ((0, 0, 0, 0), (0, 0), (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)),
            ((f, f, f, f), (f, f), (0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd)),
            ((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), (0xa4093822, 0x299f31d0),
             (0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1))):
        assert tuple(R.philox([np.array([x]) for x in ctr], key)[:, 0]) == want


def test_mask_statistics_of_the_reference():
    """Kept shares and neighbouring pairs are those of independent draws (six
    standard deviations)."""
    n = 1 << 18
    for p in (0.1, 0.5):
        k = R.keep(7, 3, 11, n, p)
        q = 1 - R.threshold(p) / 65536
        assert abs(k.mean() - q) < 6 * np.sqrt(q * (1 - q) / n)
        assert abs((k[1:] & k[:-1]).mean() - q * q) < 6 * np.sqrt(q * q * (1 - q * q) * 3 / n)
    assert R.keep(7, 3, 0, 99, 0.0).all() and not R.keep(7, 3, 0, 99, 1.0).any()


def test_reference_gradients_are_those_of_differences():
    """The formulas' gradients against central differences in 64 bits: the
    error of (f(x + h) - f(x - h)) / 2h is h^2 / 6 times a third derivative of
    order one, and 2^-53 / h."""
    rng = np.random.default_rng(1)
    x, h = rng.normal(size=(7, 5)), 1e-4
    index = np.argsort(-x, 1)[:, :2]
    mask = np.array([1, 1, 0, 1, 1, 1, 0])
    counts, _ = R.balance_stats(x, index, mask)

    def loss(z):
        return R.balance_loss(counts, R.balance_stats(z, index, mask)[1], 2, 0.7, 0.3)[0]
    g = R.balance_grad(x, mask, counts, 2, 0.7, 0.3)
    for i in np.ndindex(x.shape):
        e = np.zeros_like(x)
        e[i] = h
        assert abs((loss(x + e) - loss(x - e)) / (2 * h) - g[i]) < 1e-7
    old = -rng.random((4, 6)) * 2
    logp, ref = old + rng.normal(size=old.shape) * 0.4, old + rng.normal(size=old.shape)
    adv = rng.normal(size=(4, 1)) + np.zeros((4, 6))
    m = (np.arange(6) < np.array([[6], [0], [3], [1]])).astype(np.uint8)
    for per_sequence in (False, True):
        def policy(z):
            pg, kl, cut, _, _ = R.policy_terms(z, old, adv, ref, 0.2, 0.3)
            sums, counts, _, _ = R.policy_stats(pg, kl, cut, m, per_sequence)
            return R.policy_loss(sums, counts, per_sequence, 0.1)[0]
        pg, kl, cut, dpg, dkl = R.policy_terms(logp, old, adv, ref, 0.2, 0.3)
        _, counts, rows, _ = R.policy_stats(pg, kl, cut, m, per_sequence)
        g = R.policy_grad(dpg, dkl, m, rows, counts, per_sequence, 0.1)
        for i in np.ndindex(logp.shape):
            e = np.zeros_like(logp)
            e[i] = h
            # away from the corner of the clip, where there is no derivative
            if min(abs(logp[i] - old[i] - np.log1p(0.3)), abs(logp[i] - old[i] - np.log1p(-0.2))) > h:
                assert abs((policy(logp + e) - policy(logp - e)) / (2 * h) - g[i]) < 1e-6


def test_parameter_structs_match_the_header(tmp_path):
    """What Python packs is what a C program reads in the header's structs,
    field by field."""
    pairs = (("dropout", _lib.DROPOUT_FIELDS, _lib.DropoutParams,
              (10, 9, 3 << 40, 5 << 41, 0.125, 2 ** 64 - 7, 2 ** 63 + 9, 77, PTR)),
             ("balance", _lib.BALANCE_FIELDS, _lib.BalanceParams,
              (8, 6, 1 << 50, 2, 3, 4, 5 << 40, 6, 0.5, -0.25)),
             ("policy", _lib.POLICY_FIELDS, _lib.PolicyParams,
              (9, 1, 0, 1 << 33, 2 << 34, 3 << 35, 0.25, 4.5, -8.0)))
    lines, want = [], []
    for name, fields, pack, values in pairs:
        lines.append(f'{{ ucg_builtin_dev_{name}_params_t q; if (fread(&q, sizeof(q), 1, stdin) != 1) return 1;')
        lines += [f'printf("%.17g\\n", (double)(uintptr_t)q.{f});' if f == "rng" else
                  f'printf("%.17g\\n", (double)q.{f});' for f in fields]
        lines.append("}")
        want.append((pack(*values), values))
    lines.append("return getchar() == EOF ? 0 : 2;")
    src = tmp_path / "p.c"
    src.write_text('#include <stdio.h>\n#include "ucg_builtin_dev.h"\nint main(void) {\n' +
                   "\n".join(lines) + "\n}\n")
    exe = str(tmp_path / "p")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe], check=True)
    p = subprocess.run([exe], input=b"".join(w for w, _ in want), check=True, capture_output=True)
    assert [float(x) for x in p.stdout.split()] == [float(x) for _, v in want for x in v]


def refused(fn, status, why, *args):
    """The call (with no context, so that nothing could run) is refused with
    `status`, for the reason `why`."""
    assert getattr(_lib.dev(), fn)(None, *args) == status
    assert why in _lib.last_error(), _lib.last_error()


def srcs_of(*ptrs):
    return _lib.addresses(ptrs)


def test_sum_dropout_refusals():
    def P(dt="float32", out="float32", rows=4, cols=8, p=0.1, offset=0, rng=None):
        return _lib.DropoutParams(DT[dt], DT[out], rows, cols, p, 1, 2, offset, rng or 0)
    f, s = "ucg_builtin_dev_sum_dropout", srcs_of(PTR)

    def bad(why, q, dst=2 * PTR, srcs=s, n=1, bias=None, res=None, status=INVALID):
        refused(f, status, why, q, dst, srcs, n, bias, res)
    bad("params is NULL", None)
    for dt, out in (("float64", "float64"), ("int32", "int32"), ("float32", "bfloat16"),
                    ("bfloat16", "float16"), ("bfloat16", "float64")):
        bad("dt must be", P(dt, out), status=UNSUPPORTED)
    for p in (-0.1, 1.0001, float("nan"), float("inf")):
        bad("p must be in [0, 1]", P(p=p))
    bad("does not fit", P(rows=1 << 40, cols=1 << 40))
    bad("offset", P(offset=(1 << 63) - 16))
    bad("offset", P(offset=(1 << 64) - 16))
    bad("misaligned rng", P(rng=PTR + 4))
    bad("nsrc must be", P(), n=0)
    bad("nsrc must be", P(), n=17)
    bad("nsrc must be", P(), srcs=None)
    bad("NULL dst", P(), dst=None)
    bad("misaligned", P(), dst=2 * PTR + 2)
    bad("misaligned", P(), res=2 * PTR + 1)
    bad("misaligned", P(), bias=PTR + 2)
    bad("source", P(), srcs=srcs_of(PTR, None), n=2)
    bad("source", P(), srcs=srcs_of(PTR + 1))
    bad("overlaps a source", P(), dst=PTR + 4)
    bad("overlaps a source", P("bfloat16", "float32"), dst=PTR)
    bad("overlaps the residual", P(), res=2 * PTR + 4)
    bad("overlaps the residual, the bias or rng", P(), bias=2 * PTR + 64)
    bad("overlaps the residual, the bias or rng", P(rng=2 * PTR + 64))
    # what is allowed comes as far as the missing context
    bad("ctx is NULL", P(), dst=PTR)
    bad("ctx is NULL", P(), res=2 * PTR)
    bad("ctx is NULL", P(rows=0), dst=None, srcs=srcs_of(None))


def test_sum_dropout_grad_refusals():
    f = "ucg_builtin_dev_sum_dropout_grad"

    def P(dt="float32", out="float32", rows=4000, cols=8, p=0.1):
        return _lib.DropoutParams(DT[dt], DT[out], rows, cols, p, 1, 2, 0, 0)
    need = xucg_amd.DevContext.sum_dropout_grad_workspace(4000, 8)
    assert need > 0 and need % 16 == 0
    assert xucg_amd.DevContext.sum_dropout_grad_workspace(0, 8) == 0
    assert xucg_amd.DevContext.sum_dropout_grad_workspace(4000, 0) == 0
    M = 1 << 30

    def bad(why, q, dsrc=2 * M, grad=3 * M, dbias=4 * M, ws=5 * M, n=need, status=INVALID):
        refused(f, status, why, q, dsrc, grad, dbias, ws, n)
    bad("params is NULL", None)
    bad("dt must be", P("int8", "int8"), status=UNSUPPORTED)
    bad("p must be", P(p=2))
    bad("NULL or misaligned", P(), dsrc=None)
    bad("NULL or misaligned", P(), grad=3 * M + 1)
    bad("misaligned dbias", P(), dbias=4 * M + 2)
    bad("misaligned dbias or workspace", P(), ws=5 * M + 8)
    bad("workspace is missing", P(), ws=None)
    bad("too small", P(), n=need - 1)
    bad("2^27 columns", P(rows=1, cols=(1 << 27) + 1))
    bad("overlapping", P(), dsrc=3 * M + 16)
    bad("overlapping", P("bfloat16", "float32"), dsrc=3 * M)
    bad("overlapping", P(), dbias=3 * M + 16)
    bad("overlapping", P(), ws=2 * M + 16)
    bad("overlapping", P(), ws=4 * M - 16)
    bad("ctx is NULL", P(), dsrc=3 * M)
    bad("ctx is NULL", P(), dbias=None, ws=None, n=0)


def test_balance_refusals():
    def P(dt="float32", idt="int64", tokens=100, experts=8, topk=2, ld=0, ldi=0, ldo=0, a=0.1,
          z=0.0):
        return _lib.BalanceParams(DT[dt], DT[idt], tokens, experts, topk, ld, ldi, ldo, a, z)
    M = 1 << 30
    need = xucg_amd.DevContext.balance_workspace(1 << 20, 8)
    assert need > 0 and xucg_amd.DevContext.balance_workspace(0, 8) == 0

    def bad(why, q, logits=M, index=2 * M, mask=None, counts=3 * M, sums=4 * M, loss=None, ws=None,
            n=0, status=INVALID):
        refused("ucg_builtin_dev_balance", status, why, q, logits, index, mask, counts, sums, loss,
                ws, n)
    bad("params is NULL", None)
    bad("dt must be", P("float64"), status=UNSUPPORTED)
    bad("index_dt", P(idt="int16"), status=UNSUPPORTED)
    for e, k in ((0, 1), (1025, 1), (8, 0), (8, 9)):
        bad("experts must be", P(experts=e, topk=k))
    bad("coefficients", P(a=float("nan")))
    bad("coefficients", P(z=float("inf")))
    bad("row step", P(ld=7))
    bad("row step", P(ldi=1))
    bad("row step", P(ldo=7))
    bad("does not fit", P(tokens=1 << 62))
    bad("NULL buffer", P(), logits=None)
    bad("NULL buffer", P(), counts=None)
    bad("misaligned", P(), index=2 * M + 4)
    bad("misaligned", P(), counts=3 * M + 4)
    bad("workspace", P(tokens=1 << 20))
    bad("workspace", P(tokens=1 << 20), ws=5 * M, n=need - 1)
    bad("overlapping", P(), counts=M)
    bad("overlapping", P(), sums=2 * M)
    bad("overlapping", P(), sums=3 * M + 64)
    bad("overlapping", P(), loss=4 * M)
    bad("overlapping", P(), mask=3 * M)
    bad("overlapping", P(tokens=1 << 20), ws=4 * M, n=need)
    bad("ctx is NULL", P(tokens=1 << 20), ws=5 * M, n=need)
    bad("ctx is NULL", P(tokens=0), logits=None, index=None)
    refused("ucg_builtin_dev_balance_loss", INVALID, "NULL", P(), None, M, M)
    refused("ucg_builtin_dev_balance_loss", INVALID, "overlapping", P(), M, 2 * M, M)
    refused("ucg_builtin_dev_balance_loss", INVALID, "ctx is NULL", P(), M, 2 * M, 3 * M)

    def badg(why, q, logits=M, mask=None, counts=3 * M, base=None, g=None, d=5 * M, status=INVALID):
        refused("ucg_builtin_dev_balance_grad", status, why, q, logits, mask, counts, base, g, d)
    badg("NULL buffer", P(), d=None)
    badg("misaligned", P(), d=5 * M + 2)
    badg("overlaps", P(), d=M + 32)
    badg("overlaps", P(ldo=9), d=M)
    badg("overlaps", P(), base=5 * M + 32)
    badg("overlaps", P(), d=3 * M)
    badg("overlaps", P(), mask=5 * M)
    badg("ctx is NULL", P(), d=M)
    badg("ctx is NULL", P(), base=5 * M)


def test_policy_refusals():
    def P(dt="float32", rows=4, cols=9, ld=0, low=0.2, high=0.2, kl=0.1, per_row=0, seq=0):
        return _lib.PolicyParams(DT[dt], per_row, seq, rows, cols, ld, low, high, kl)
    M = 1 << 30
    need = xucg_amd.DevContext.policy_workspace(4, 9)

    def bad(why, q, logp=M, old=2 * M, ref=None, adv=3 * M, mask=None, sums=4 * M, counts=5 * M,
            rt=None, loss=None, ws=6 * M, n=need, status=INVALID):
        refused("ucg_builtin_dev_policy", status, why, q, logp, old, ref, adv, mask, sums, counts,
                rt, loss, ws, n)
    bad("params is NULL", None)
    bad("dt must be", P("float64"), status=UNSUPPORTED)
    for k in (dict(low=-0.1), dict(low=1.1), dict(high=-0.1), dict(high=float("inf")),
              dict(kl=float("nan")), dict(low=float("nan"))):
        bad("clip_low", P(**k))
    bad("row step", P(ld=8))
    bad("does not fit", P(rows=1 << 47, cols=1 << 30))
    bad("does not fit", P(rows=1 << 50, cols=0))
    bad("does not fit", P(cols=1 << 31))
    bad("NULL buffer", P(), adv=None)
    bad("NULL buffer", P(), sums=None)
    bad("misaligned", P(), logp=M + 2)
    bad("misaligned", P(), counts=5 * M + 4)
    bad("workspace", P(), ws=None)
    bad("workspace", P(), n=need - 1)
    bad("overlapping", P(), sums=M)
    bad("overlapping", P(), rt=5 * M + 16)
    bad("overlapping", P(per_row=1), ws=3 * M)
    bad("overlapping", P(), loss=4 * M)
    bad("ctx is NULL", P())
    refused("ucg_builtin_dev_policy_loss", INVALID, "NULL", P(), M, M, None)
    refused("ucg_builtin_dev_policy_loss", INVALID, "overlapping", P(), M, 2 * M, M)

    def badg(why, q, logp=M, old=2 * M, ref=None, adv=3 * M, mask=None, rt=None, counts=5 * M,
             g=None, d=7 * M, status=INVALID):
        refused("ucg_builtin_dev_policy_grad", status, why, q, logp, old, ref, adv, mask, rt,
                counts, g, d)
    badg("row_tokens", P(seq=1))
    badg("NULL buffer", P(), d=None)
    badg("misaligned", P(), g=M + 2)
    badg("overlaps", P(), d=M + 4)
    badg("overlaps", P(), d=3 * M)
    badg("overlaps", P(), d=5 * M)
    badg("overlaps", P(), mask=7 * M)
    badg("ctx is NULL", P(), d=M)
    badg("ctx is NULL", P(), d=2 * M)


def test_kernels_keep_off_scratch_and_packed_fp32():
    """No kernel of dev_train.hip spills or indexes into scratch memory, and none
    holds a packed fp32 instruction (read from the built object)."""
    import re
    llvm, obj = "/opt/rocm/lib/llvm/bin", os.path.join(ROOT, "xucg_amd", "csrc", "_obj", "dev_train.o")
    if not os.path.exists(obj) or not os.path.exists(f"{llvm}/clang-offload-bundler"):
        pytest.skip("the device object is not built here")
    import tempfile
    with tempfile.TemporaryDirectory() as d:
        fb, co = os.path.join(d, "fb"), os.path.join(d, "co")
        subprocess.run([f"{llvm}/llvm-objcopy", f"--dump-section=.hip_fatbin={fb}", obj,
                        os.path.join(d, "junk")], check=True, capture_output=True)
        subprocess.run([f"{llvm}/clang-offload-bundler", "--type=o", "--unbundle",
                        "--targets=hipv4-amdgcn-amd-amdhsa--gfx950", f"--input={fb}", f"--output={co}"],
                       check=True, capture_output=True)
        notes = subprocess.run([f"{llvm}/llvm-readelf", "--notes", co], check=True, capture_output=True,
                               text=True).stdout
        code = subprocess.run([f"{llvm}/llvm-objdump", "-d", "--no-show-raw-insn", co], check=True,
                              capture_output=True, text=True).stdout
    scratch = [int(x) for x in re.findall(r"\.private_segment_fixed_size:\s+(\d+)", notes)]
    assert len(scratch) > 100 and not any(scratch)
    assert not re.search(r"v_pk_(add|mul|fma)_f32", code) and "v_bitop3_b32" in code


def test_python_refusals():
    """What is no device memory, too small a buffer, numbers that no size is."""
    ctx = xucg_amd.DevContext.__new__(xucg_amd.DevContext)   # no GPU is needed to refuse
    ctx.handle, ctx.device = None, 0
    buf = xucg_amd.DevBuffer.__new__(xucg_amd.DevBuffer)
    buf.ptr, buf.nbytes = PTR, 4 * 32
    x = np.zeros(32, np.float32)
    with pytest.raises(TypeError, match="dst"):
        ctx.sum_dropout("float32", x, [PTR], 4, 8, 0.1, 1)
    with pytest.raises(TypeError, match="srcs"):
        ctx.sum_dropout("float32", PTR, [x], 4, 8, 0.1, 1)
    with pytest.raises(ValueError, match="dst"):
        ctx.sum_dropout("float32", buf, [2 * PTR], 4, 9, 0.1, 1)
    with pytest.raises(ValueError, match="logits"):
        ctx.balance("float32", buf, PTR, 4, 8, 2, PTR, PTR, ld=9)
    for bad in (dict(rows=-1), dict(p="x"), dict(seed=-1), dict(rows=1.5)):
        kw = dict(dict(rows=4, p=0.1, seed=1), **bad)
        with pytest.raises((ValueError, TypeError)):
            ctx.sum_dropout("float32", PTR, [2 * PTR], kw["rows"], 8, kw["p"], kw["seed"])
    with pytest.raises(xucg_amd.UcsError, match="NULL or misaligned source"):
        ctx.sum_dropout("float32", PTR, [None], 4, 8, 0.1, 1)
    with pytest.raises(xucg_amd.UcsError, match="nsrc must be"):
        ctx.sum_dropout("float32", PTR, [2 * PTR] * 17, 4, 8, 0.1, 1)
    with pytest.raises(KeyError):
        ctx.sum_dropout("float31", PTR, [2 * PTR], 4, 8, 0.1, 1)
    buf.ptr = None                       # nothing to free


def test_row_bounds_cover():
    for rows in (0, 1, 7, 64, 1001):
        for world in (1, 2, 3, 8):
            b = [G.row_bounds(rows, world, r) for r in range(world)]
            assert b[0][0] == 0 and b[-1][1] == rows
            assert all(x[1] == y[0] for x, y in zip(b, b[1:]))
            assert max(y - x for x, y in b) - min(y - x for x, y in b) <= 1
    with pytest.raises(ValueError):
        G.row_bounds(4, 2, 2)


# ---- GPU ---------------------------------------------------------------------------
GUARD = 64            # bytes before and behind every array, which stay as they were


class Arr:
    """A device array between guards, `shift` elements past a 256-byte line."""

    def __init__(self, ctx, x, shift=0):
        self.x = np.ascontiguousarray(x)
        self.at = 256 + shift * self.x.itemsize
        self.buf = ctx.alloc(self.at + self.x.nbytes + GUARD)
        self.whole = np.full(self.at + self.x.nbytes + GUARD, 0xA5, np.uint8)
        self.whole[self.at:self.at + self.x.nbytes] = self.x.reshape(-1).view(np.uint8)
        self.buf.upload(self.whole)
        self.ptr = self.buf.ptr + self.at

    def get(self):
        """its values; the guards must be untouched"""
        w = self.buf.download(np.uint8, self.whole.size)
        end = self.at + self.x.nbytes
        assert (w[:self.at] == 0xA5).all() and (w[end:] == 0xA5).all(), "written outside"
        return w[self.at:end].copy().view(self.x.dtype).reshape(self.x.shape)


def ptr(a):
    return None if a is None else a.ptr


def gpu(f):
    return pytest.mark.gpu(f)


def drop_inputs(rng, dt, out_dt, rows, cols, nsrc, with_bias=True, with_res=True):
    srcs = [R.to_storage(rng.normal(size=(rows, cols)), dt) for _ in range(nsrc)]
    bias = R.to_storage(rng.normal(size=cols), dt) if with_bias else None
    res = R.to_storage(rng.normal(size=(rows, cols)), out_dt) if with_res else None
    return srcs, bias, res


def val(x, dt):
    return None if x is None else R.from_storage(x, dt)


def check_drop(got, srcs, bias, res, dt, out_dt, keep, p):
    """nsrc - 1 sums, the bias, the scale and its own rounding, the residual,
    then the output's type"""
    want, size = R.sum_dropout([val(s, dt) for s in srcs], val(bias, dt), val(res, out_dt),
                               keep.reshape(got.shape), p)
    tol = (len(srcs) + 4) * U * size * 1.01
    tol = tol + R.EPS[out_dt] * (np.abs(want) + tol) + R.LEAST[out_dt]
    off = np.abs(val(got, out_dt) - want)
    assert (off <= tol).all(), (off / np.maximum(tol, 1e-300)).max()


DROP_CASES = [
    # rows, cols, nsrc, p, offset, shift of every array in elements
    (1, 1, 1, 0.1, 0, 0), (1, 1, 2, 0.5, 3, 1), (5, 1, 1, 0.5, 0, 0), (1, 7, 3, 0.5, 0, 0),
    (3, 8, 1, 0.1, 8, 0), (5, 13, 2, 0.25, 5, 1), (2, 64, 4, 0.1, 0, 0), (64, 96, 8, 0.1, 1 << 33, 0),
    (33, 1023, 2, 0.25, (1 << 35) + 5, 3), (128, 1000, 16, 0.5, 7, 0), (16, 257, 5, 0.9, 2, 1),
    (9, 40, 7, 0.0, 1, 0), (9, 40, 1, 1.0, 0, 0), (700, 3, 1, 0.5, 4, 1), (3, 4096, 1, 2 ** -17, 0, 0),
]


@gpu
@pytest.mark.parametrize("dt,out_dt", [("float32", "float32"), ("bfloat16", "bfloat16"),
                                       ("float16", "float16"), ("bfloat16", "float32"),
                                       ("float16", "float32")])
@pytest.mark.parametrize("rows,cols,nsrc,p,offset,shift", DROP_CASES)
def test_sum_dropout(dev_ctx, dt, out_dt, rows, cols, nsrc, p, offset, shift):
    rng = np.random.default_rng(rows * 1000 + cols)
    seed, tag = 0x123456789ABCDEF0 + rows, (5 << 32) + cols
    keep = R.keep(seed, tag, offset, rows * cols, p)
    for with_bias, with_res in ((True, True), (False, False), (True, False), (False, True)):
        srcs, bias, res = drop_inputs(rng, dt, out_dt, rows, cols, nsrc, with_bias, with_res)
        a = [Arr(dev_ctx, s, shift) for s in srcs]
        b, r = [x if x is None else Arr(dev_ctx, x, shift) for x in (bias, res)]
        out = Arr(dev_ctx, np.zeros((rows, cols), R.STORAGE[out_dt]), shift)
        dev_ctx.sum_dropout(dt, out.ptr, [s.ptr for s in a], rows, cols, p, seed, tag=tag,
                            offset=offset, bias=ptr(b), residual=ptr(r), out_dt=out_dt)
        dev_ctx.sync()
        check_drop(out.get(), srcs, bias, res, dt, out_dt, keep, p)
        if res is None:
            assert (val(out.get(), out_dt).reshape(-1)[~keep] == 0).all()
        else:                                 # a dropped element is the residual, bit for bit
            assert (out.get().reshape(-1)[~keep] == res.reshape(-1)[~keep]).all()


@gpu
@pytest.mark.parametrize("dt", DTS)
def test_sum_dropout_drops_what_is_not_finite(dev_ctx, dt):
    rows, cols, p = 40, 33, 0.5
    keep = R.keep(1, 2, 0, rows * cols, p).reshape(rows, cols)
    x = np.ones((rows, cols))
    x[~keep] = np.nan
    x[0] = np.where(keep[0], 1, np.inf)
    a, out = Arr(dev_ctx, R.to_storage(x, dt)), Arr(dev_ctx, R.to_storage(np.full((rows, cols), 7.0), dt))
    dev_ctx.sum_dropout(dt, out.ptr, [a.ptr], rows, cols, p, 1, tag=2)
    dev_ctx.sync()
    assert (val(out.get(), dt) == np.where(keep, 2.0, 0.0)).all()


@gpu
def test_sum_dropout_is_the_combine_without_dropout(dev_ctx):
    """fp32, p = 0: the bits of reduce_multi (2^k operands) and reduce_tree."""
    rng, n = np.random.default_rng(3), 10007
    for nsrc in (1, 2, 3, 4, 5, 8, 12, 16):
        a = [Arr(dev_ctx, rng.normal(size=n).astype(np.float32)) for _ in range(nsrc)]
        out, want = [Arr(dev_ctx, np.zeros(n, np.float32)) for _ in range(2)]
        dev_ctx.sum_dropout("float32", out.ptr, [s.ptr for s in a], 1, n, 0.0, 1)
        ptrs = [s.ptr for s in a]
        rc = (dev_ctx.reduce_multi("sum", "float32", want.ptr, ptrs, 0, n)
              if nsrc & (nsrc - 1) == 0 else dev_ctx.reduce_tree("sum", "float32", want.ptr, ptrs, n))
        assert rc == 0
        dev_ctx.sync()
        assert (out.get().view(np.uint32) == want.get().view(np.uint32)).all(), nsrc


@gpu
@pytest.mark.parametrize("dt", DTS)
def test_sum_dropout_of_shards_is_that_of_the_whole(dev_ctx, dt):
    """Rows cut anywhere: the same bits; in place on the residual and on a source."""
    rows, cols, p, offset = 37, 75, 0.3, 1 << 32
    rng = np.random.default_rng(4)
    srcs, bias, res = drop_inputs(rng, dt, dt, rows, cols, 2)
    a, b = [Arr(dev_ctx, s) for s in srcs], Arr(dev_ctx, bias)
    out = Arr(dev_ctx, np.zeros_like(res))
    r = Arr(dev_ctx, res)
    dev_ctx.sum_dropout(dt, out.ptr, [s.ptr for s in a], rows, cols, p, 9, offset=offset,
                        bias=b.ptr, residual=r.ptr)
    dev_ctx.sync()
    whole = out.get()
    size = res.itemsize
    for lo, hi in ((0, 1), (1, 12), (12, 37)):
        at = lo * cols * size
        dev_ctx.sum_dropout(dt, r.ptr + at, [s.ptr + at for s in a], hi - lo, cols, p, 9,
                            offset=offset + lo * cols, bias=b.ptr, residual=r.ptr + at)
    dev_ctx.sync()
    assert (r.get() == whole).all()
    # in place on a source that comes twice
    dev_ctx.sum_dropout(dt, out.ptr, [a[0].ptr, a[0].ptr], rows, cols, p, 9, bias=b.ptr)
    dev_ctx.sum_dropout(dt, a[0].ptr, [a[0].ptr, a[0].ptr], rows, cols, p, 9, bias=b.ptr)
    dev_ctx.sync()
    assert (a[0].get() == out.get()).all()


@gpu
def test_sum_dropout_state_in_device_memory(dev_ctx):
    x = np.ones((5, 100), np.float32)
    a, out = Arr(dev_ctx, x), Arr(dev_ctx, x * 0)
    state = Arr(dev_ctx, np.array([0xFEDCBA9876543210, 77], np.uint64))
    dev_ctx.sum_dropout("float32", out.ptr, [a.ptr], 5, 100, 0.5, 1, tag=2, rng=state.ptr)
    dev_ctx.sync()
    keep = R.keep(0xFEDCBA9876543210, 77, 0, 500, 0.5).reshape(5, 100)
    assert (out.get() == np.where(keep, 2, 0)).all()


GRAD_CASES = [(1, 1, 0), (1, 8, 0), (3, 5, 3), (300, 1, 1), (5, 64, 0), (257, 96, 8), (64, 1023, 5),
              (1000, 33, 1 << 34), (9, 2050, 7), (700, 256, 4), (2049, 8, 0), (0, 16, 0)]


@gpu
@pytest.mark.parametrize("dt,grad_dt", [("float32", "float32"), ("bfloat16", "bfloat16"),
                                        ("float16", "float16"), ("bfloat16", "float32"),
                                        ("float16", "float32")])
@pytest.mark.parametrize("rows,cols,offset", GRAD_CASES)
def test_sum_dropout_grad(dev_ctx, dt, grad_dt, rows, cols, offset):
    """dsrc: the scale, its own rounding, the type's. dbias: as many sums in
    fp32 as there are rows at most, the join's and the last rounding."""
    rng = np.random.default_rng(rows + cols)
    p, seed, tag = 0.3, 99, 1 << 40
    g = R.to_storage(rng.normal(size=(rows, cols)), grad_dt)
    mask = R.keep(seed, tag, offset, rows * cols, p).reshape(rows, cols)
    d64 = np.where(mask, val(g, grad_dt) * R.scale(p), 0.0)
    ga = Arr(dev_ctx, g, 1)
    for with_bias in (True, False):
        d = Arr(dev_ctx, np.ones((rows, cols), R.STORAGE[dt]), 1)
        db = Arr(dev_ctx, np.ones(cols, np.float32), 1) if with_bias else None
        ws = dev_ctx.alloc(max(16, dev_ctx.sum_dropout_grad_workspace(rows, cols)))
        ws.upload(np.full(ws.nbytes, 0xFF, np.uint8))       # NaN: nothing of it may be used
        dev_ctx.sum_dropout_grad(dt, d.ptr, ga.ptr, rows, cols, p, seed, tag=tag, offset=offset,
                                 dbias=ptr(db), grad_dt=grad_dt, workspace=ws)
        dev_ctx.sync()
        off = np.abs(val(d.get(), dt) - d64)
        assert (off <= (2 * U + R.EPS[dt] * 1.01) * np.abs(d64) + R.LEAST[dt]).all()
        if with_bias:
            got = db.get()
            off = np.abs(got.astype(np.float64) - d64.sum(0))
            assert (off <= (rows + 6) * U * np.abs(d64).sum(0) + 1e-30).all()
            dev_ctx.sum_dropout_grad(dt, d.ptr, ga.ptr, rows, cols, p, seed, tag=tag, offset=offset,
                                     dbias=db.ptr, grad_dt=grad_dt, workspace=ws)
            dev_ctx.sync()
            assert (db.get().view(np.uint32) == got.view(np.uint32)).all()   # the same bits again


@gpu
def test_sum_dropout_grad_is_that_of_differences(dev_ctx):
    """The operator is linear in its sources and its bias: the differences of
    the forward kernel's outputs along v are <grad, f(x + v) - f(x)>."""
    rows, cols, p = 30, 50, 0.4
    rng = np.random.default_rng(8)
    x, v, g = (rng.integers(-8, 9, (rows, cols)).astype(np.float32) for _ in range(3))
    b, w = (rng.integers(-8, 9, cols).astype(np.float32) for _ in range(2))
    xa, ba, va, wa, ga = (Arr(dev_ctx, t) for t in (x, b, x + v, b + w, g))
    f0, f1, d = (Arr(dev_ctx, np.zeros_like(x)) for _ in range(3))
    db = Arr(dev_ctx, np.zeros(cols, np.float32))
    ws = dev_ctx.alloc(max(16, dev_ctx.sum_dropout_grad_workspace(rows, cols)))
    dev_ctx.sum_dropout("float32", f0.ptr, [xa.ptr], rows, cols, p, 5, bias=ba.ptr)
    dev_ctx.sum_dropout("float32", f1.ptr, [va.ptr], rows, cols, p, 5, bias=wa.ptr)
    dev_ctx.sum_dropout_grad("float32", d.ptr, ga.ptr, rows, cols, p, 5, dbias=db.ptr, workspace=ws)
    dev_ctx.sync()
    n = rows * cols
    f = f1.get().astype(np.float64) - f0.get()
    lhs = (g * f).sum()
    rhs = (d.get().astype(np.float64) * v).sum() + (db.get().astype(np.float64) * w).sum()
    # every value is a small whole number times the scale (64 * 2 at most)
    assert abs(lhs - rhs) <= 4 * U * n * 8 * 32 * R.scale(p)


# ---- balance -----------------------------------------------------------------------
def balance_bounds(x, mask):
    """(relative error of a probability, absolute one of a log sum exp): the
    difference to the maximum, its scaling and the scale (three roundings of
    the distance D), 2^-23 of exp2, E sums, the quotient, the product"""
    live = np.ones(len(x), bool) if mask is None else mask != 0
    xf = np.where(np.isfinite(x[live]) & (np.abs(x[live]) < 1e30), x[live], 0)
    spread = (xf.max(1) - xf.min(1)).max() if xf.size else 0.0
    e = x.shape[1]
    rel = (6 * spread + e + 10) * U
    most = np.abs(xf).max() + np.log(e) if xf.size else 0.0
    return rel, (3 * spread + e + 8 + 4 * np.log(e) + 2 * most) * U


def check_balance(counts, sums, x, index, mask):
    wc, ws = R.balance_stats(x, index, mask)
    assert (counts == wc).all()
    rel, dl = balance_bounds(x, mask)
    e, n = x.shape[1], int(wc[-1])
    off = np.abs(sums.astype(np.float64) - ws)
    assert (off[:e] <= (rel + (n + 4) * U) * ws[:e] + 1e-30).all(), (off[:e] / ws[:e]).max()
    assert off[e] <= 2 * dl * np.sqrt(n * ws[e]) + n * dl * dl + (n + 4) * U * ws[e] + 1e-30
    return wc, ws


def run_balance(ctx, dt, x, index, mask, ld=0, ldi=0, coef=0.02, z=0.003, shift=0):
    t, e = x.shape
    k = index.shape[1]
    wide = np.full((t, ld or e), np.nan)
    wide[:, :e] = x
    wide_i = np.full((t, ldi or k), -7, index.dtype)
    wide_i[:, :k] = index
    la = Arr(ctx, R.to_storage(wide, dt), shift)
    ia, ma = Arr(ctx, wide_i, shift), None if mask is None else Arr(ctx, mask, shift)
    c, s = Arr(ctx, np.full(e + 1, -1, np.int64)), Arr(ctx, np.full(e + 1, np.nan, np.float32))
    loss = Arr(ctx, np.full(3, np.nan, np.float32))
    ws = ctx.alloc(max(16, ctx.balance_workspace(t, e)))
    ws.upload(np.full(ws.nbytes, 0xFF, np.uint8))
    ctx.balance(dt, la.ptr, ia.ptr, t, e, k, c.ptr, s.ptr, mask=ptr(ma), loss=loss.ptr,
                balance_coef=coef, z_coef=z, index_dt=str(index.dtype), ld=ld, ld_index=ldi,
                workspace=ws)
    ctx.sync()
    return la, ma, c, s, loss


def balance_inputs(rng, dt, t, e, k, idt, mask):
    x = R.from_storage(R.to_storage(rng.normal(size=(t, e)) * 2 + rng.normal(size=e), dt), dt)
    index = np.argsort(-x, 1, kind="stable")[:, :k].astype(idt)
    m = {"none": None, "all": np.zeros(t, np.uint8),
         "some": (rng.random(t) < 0.7).astype(np.uint8) * 255}[mask]
    return x, index, m


BALANCE_CASES = [(1, 1, 1), (1, 8, 2), (3, 2, 1), (64, 3, 3), (65, 8, 2), (127, 16, 4), (130, 60, 6),
                 (1000, 64, 8), (257, 100, 1), (300, 160, 6), (1025, 256, 8), (70, 257, 3),
                 (33, 512, 8), (40, 600, 2), (20, 1000, 5), (19, 1024, 1024), (40000, 8, 2), (0, 8, 2)]


@gpu
@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("t,e,k", BALANCE_CASES)
def test_balance(dev_ctx, dt, t, e, k):
    """Counts exact, sums and loss, then the gradient: p (c - p.c) with both
    factors' errors, c less a mean that the p cancel."""
    rng = np.random.default_rng(t * 7 + e)
    coef, z, g = 0.02, 0.003, 1.75
    for i, mask in enumerate(("none", "some", "all")):
        x, index, m = balance_inputs(rng, dt, t, e, k, [np.int64, np.int32][i % 2], mask)
        ld, ldi, shift = [(0, 0, 0), (e + 3, k + 2, 1), (e + 8, k, 0)][i]
        la, ma, c, s, loss = run_balance(dev_ctx, dt, x, index, m, ld, ldi, coef, z, shift)
        counts, sums = c.get(), s.get()
        wc, ws = check_balance(counts, sums, x, index, m)
        rel, dl = balance_bounds(x, m)
        n = int(wc[-1])
        want = R.balance_loss(wc, ws, k, coef, z)
        tol_b = (rel + (n + 8) * U) * abs(want[1]) + 1e-30
        tol_z = (2 * dl * np.sqrt(n * ws[e]) + n * dl * dl) * z / max(n, 1) + (n + 8) * U * want[2] + 1e-30
        assert (np.abs(loss.get() - want) <= [tol_b + tol_z, tol_b, tol_z]).all()
        # the gradient, with a base and without, of the counts of a larger group
        group = counts * 3
        gc, gl = Arr(dev_ctx, group), Arr(dev_ctx, np.array([g], np.float32))
        base = R.to_storage(rng.normal(size=(t, e)) * 1e-3, dt)
        want = R.balance_grad(x, m, group, k, coef, z, g)
        p, lse = R.softmax(x)
        cc = group[:e] - group[e] * k / e
        a, b = g * coef * e / (k * max(1, group[e]) ** 2.0), g * 2 * z / max(1, group[e])
        size = 2 * np.abs(cc).max(initial=0) + 1
        tol = p * (a * size * (2 * rel + (e + 8) * U) +
                   b * (dl + (rel + 5 * U) * np.abs(lse)[:, None]))
        for ba in (None, base):
            d = Arr(dev_ctx, np.zeros((t, e), R.STORAGE[dt]), shift)
            bb = None if ba is None else Arr(dev_ctx, ba, shift)
            dev_ctx.balance_grad(dt, d.ptr, la.ptr, t, e, k, gc.ptr, mask=ptr(ma), base=ptr(bb),
                                 grad_loss=gl.ptr, balance_coef=coef, z_coef=z, ld=ld)
            dev_ctx.sync()
            w = want + (0 if ba is None else R.from_storage(ba, dt))
            o = np.abs(R.from_storage(d.get(), dt) - w)
            assert (o <= tol + R.EPS[dt] * (np.abs(w) + tol) * 1.01 + U * np.abs(w) + R.LEAST[dt]).all()


@gpu
@pytest.mark.parametrize("dt", DTS)
def test_balance_odd_rows(dev_ctx, dt):
    """Rows of -inf alone, of the lowest value alone and among others, indices
    that name nobody, masked rows of NaN, and a NaN upstream gradient."""
    e, k = 12, 3
    low = {"float32": -3.4028234663852886e38, "bfloat16": -3.3895313892515355e38,
           "float16": -65504.0}[dt]
    rng = np.random.default_rng(5)
    x = R.from_storage(R.to_storage(rng.normal(size=(9, e)), dt), dt)
    x[1], x[2], x[3, 4:], x[4, :5] = -np.inf, low, low, -np.inf
    x[7] = np.nan
    index = np.stack([rng.permutation(e)[:k] for _ in range(9)]).astype(np.int64)
    index[5] = [-1, e, 1 << 40]
    mask = np.array([1, 1, 1, 1, 1, 1, 1, 0, 1], np.uint8)
    la, ma, c, s, loss = run_balance(dev_ctx, dt, x, index, mask, z=0.0)
    wc, _ = R.balance_stats(x, index, mask)
    assert (c.get() == wc).all() and wc[-1] == 8 and wc[:-1].sum() == 7 * k
    p, _ = R.softmax(x[mask != 0])
    rel, _ = balance_bounds(x, mask)
    assert (np.abs(s.get()[:e] - p.sum(0)) <= (rel + 20 * U) * p.sum(0)).all()
    want = R.balance_loss(wc, np.append(p.sum(0), 0), k, 0.02, 0.0)
    assert np.abs(loss.get() - want).max() <= (rel + 20 * U) * want[0]
    d = Arr(dev_ctx, np.zeros((9, e), R.STORAGE[dt]))
    dev_ctx.balance_grad(dt, d.ptr, la.ptr, 9, e, k, c.ptr, mask=ma.ptr, balance_coef=0.02)
    dev_ctx.sync()
    got = R.from_storage(d.get(), dt)
    assert (got[1] == 0).all() and (got[7] == 0).all() and (got[4, :5] == 0).all()
    assert np.isfinite(got).all() and np.abs(got[0]).max() > 0
    base = Arr(dev_ctx, R.to_storage(np.full((9, e), 0.5), dt))
    nan = Arr(dev_ctx, np.array([np.nan], np.float32))
    dev_ctx.balance_grad(dt, d.ptr, la.ptr, 9, e, k, c.ptr, mask=ma.ptr, base=base.ptr,
                         grad_loss=nan.ptr, balance_coef=0.02)
    dev_ctx.sync()
    got = R.from_storage(d.get(), dt)
    assert (got[7] == 0.5).all() and np.isnan(got[0]).all()


# ---- policy ------------------------------------------------------------------------
LOW, HIGH, KL = 0.2, 0.3, 0.07
POLICY_CASES = [(1, 1), (3, 1), (5, 0), (0, 5), (1, 7), (2, 64), (70, 3), (4, 200), (9, 257), (300, 33),
                (2, 2049), (3, 20001), (1, 70000), (600, 40)]


@gpu
@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("rows,cols", POLICY_CASES)
def test_policy(dev_ctx, dt, rows, cols):
    """Per token: d and its exponential (2 u of d's, 4 u), the product; kl: up
    to 40 u near the series' end, 2 |q| more; sums: 32 values of a lane, its six
    neighbours, the last rounding."""
    rng = np.random.default_rng(rows * 31 + cols)
    for i in range(4):
        per_row, seq, with_ref, masked = i % 2 == 0, i >= 2, i != 1, i != 0
        ld = cols + [0, 5, 8, 0][i]
        shape = (rows, cols)
        old = R.to_storage(-rng.random(shape) * 3, dt)
        o64 = R.from_storage(old, dt)
        lp = R.to_storage(o64 + rng.normal(size=shape) * 0.3, dt)
        rf = R.to_storage(o64 + rng.normal(size=shape) * 0.5, dt)
        adv = rng.normal(size=(rows,) if per_row else shape).astype(np.float32)
        a64 = np.broadcast_to((adv[:, None] if per_row else adv).astype(np.float64), shape)
        mask = (rng.random(shape) < 0.6).astype(np.uint8) if masked else np.ones(shape, np.uint8)
        if masked and rows > 1:
            mask[rows // 2] = 0

        def wide(x, fill):
            w = np.full((rows, ld), fill, x.dtype)
            w[:, :cols] = x
            return w
        nan = R.to_storage(np.array([np.nan]), dt)[0]
        # masked tokens and the steps between rows hold what must not be seen
        hide = mask == 0
        bad = [np.where(hide, nan, x).astype(x.dtype) for x in (lp, old, rf)]
        la, oa, ra = (Arr(dev_ctx, wide(x, nan), i % 3) for x in bad)
        aa = Arr(dev_ctx, adv if per_row else wide(adv, np.nan), 1)
        ma = Arr(dev_ctx, wide(mask, 1), i) if masked else None
        s, c = Arr(dev_ctx, np.zeros(2, np.float32)), Arr(dev_ctx, np.zeros(3, np.int64))
        rt, loss = Arr(dev_ctx, np.full(rows, -1, np.int32)), Arr(dev_ctx, np.ones(3, np.float32))
        ws = dev_ctx.alloc(dev_ctx.policy_workspace(rows, cols))
        ws.upload(np.full(ws.nbytes, 0xFF, np.uint8))
        kw = dict(ref=ra.ptr if with_ref else None, mask=ptr(ma), row_tokens=rt.ptr,
                  adv_per_row=per_row, per_sequence=seq, clip_low=LOW, clip_high=HIGH, kl_coef=KL,
                  ld=0 if ld == cols else ld)
        dev_ctx.policy(dt, la.ptr, oa.ptr, aa.ptr, rows, cols, s.ptr, c.ptr, loss=loss.ptr,
                       workspace=ws, **kw)
        dev_ctx.sync()
        l64, r64 = R.from_storage(lp, dt), R.from_storage(rf, dt) if with_ref else None
        pg, kl, cut, dpg, dkl = R.policy_terms(l64, o64, a64, r64, LOW, HIGH)
        sums, counts, tokens, size = R.policy_stats(pg, kl, cut, mask, seq)
        assert (c.get() == counts).all() and (rt.get() == tokens).all()
        dmax = np.abs(l64 - o64).max(initial=0)
        q = np.abs(r64 - l64) if with_ref else np.zeros(shape)
        tol = np.array([(dmax + 8 + 40) * U * size[0], (80 + 2 * q.max(initial=0)) * U * size[1]])
        assert (np.abs(s.get() - sums) <= tol + 1e-30).all()
        want = R.policy_loss(sums, counts, seq, KL)
        n = max(1, counts[1] if seq else counts[0])
        t = [(tol[0] + KL * tol[1]) / n + 4 * U * (abs(want[1]) + KL * want[2]), tol[0] / n + 4 * U * abs(want[1]),
             tol[1] / n + 4 * U * want[2]]
        assert (np.abs(loss.get() - want) <= np.array(t) + 1e-30).all()
        # the gradient within a group of twice as many
        group = counts * 2
        gc, gl = Arr(dev_ctx, group.astype(np.int64)), Arr(dev_ctx, np.array([-1.5], np.float32))
        d = Arr(dev_ctx, wide(np.zeros(shape, R.STORAGE[dt]), 3))
        dev_ctx.policy_grad(dt, d.ptr, la.ptr, oa.ptr, aa.ptr, rows, cols, gc.ptr, grad_loss=gl.ptr, **kw)
        dev_ctx.sync()
        w = R.policy_grad(dpg, dkl, mask, tokens, group, seq, KL, -1.5)
        weight = np.abs(R.policy_grad(np.ones(shape), np.zeros(shape), mask, tokens, group, seq, KL, -1.5))
        e = np.maximum(np.exp(r64 - l64), 1) if with_ref else np.zeros(shape)
        t = weight * U * ((dmax + 10) * np.abs(dpg) + KL * (q + 42) * (e + q))
        got = d.get()
        off = np.abs(R.from_storage(got[:, :cols], dt) - w)
        assert (off <= t + R.EPS[dt] * (np.abs(w) + t) * 1.01 + U * np.abs(w) + R.LEAST[dt]).all()
        assert (got[:, cols:] == 3).all()            # between rows nothing is written


@gpu
@pytest.mark.parametrize("rows", [5, 3000])
@pytest.mark.parametrize("per_row", [False, True])
def test_policy_rows_without_columns_read_nothing(dev_ctx, rows, per_row):
    s, c = Arr(dev_ctx, np.ones(2, np.float32)), Arr(dev_ctx, np.ones(3, np.int64))
    rt, loss = Arr(dev_ctx, np.full(rows, -1, np.int32)), Arr(dev_ctx, np.ones(3, np.float32))
    ws = dev_ctx.alloc(dev_ctx.policy_workspace(rows, 0))
    dev_ctx.policy("bfloat16", None, None, None, rows, 0, s.ptr, c.ptr, row_tokens=rt.ptr,
                   adv_per_row=per_row, per_sequence=True, loss=loss.ptr, workspace=ws)
    dev_ctx.policy_grad("bfloat16", None, None, None, None, rows, 0, c.ptr, row_tokens=rt.ptr,
                        adv_per_row=per_row, per_sequence=True)
    dev_ctx.sync()
    assert not s.get().any() and not c.get().any() and not rt.get().any() and not loss.get().any()


@gpu
def test_policy_clip_goes_by_the_difference(dev_ctx):
    """At a limit a token is not cut, one step beyond it is; A = 0 never is.
    clip_low = 1 never cuts below."""
    up, down = np.float32(np.log1p(HIGH)), np.float32(np.log1p(-LOW))
    d = np.array([up, np.nextafter(up, np.float32(9)), down, np.nextafter(down, np.float32(-9)),
                  5, -5, 5, -5], np.float32)[None]
    adv = np.array([1, 1, -1, -1, 0, 0, -1, 1], np.float32)[None]
    la, oa, aa = Arr(dev_ctx, d), Arr(dev_ctx, d * 0), Arr(dev_ctx, adv)
    s, c, g = Arr(dev_ctx, np.zeros(2, np.float32)), Arr(dev_ctx, np.zeros(3, np.int64)), Arr(dev_ctx, d * 0)
    ws = dev_ctx.alloc(dev_ctx.policy_workspace(1, 8))
    for low, cut in ((LOW, [0, 1, 0, 1, 0, 0, 0, 0]), (1.0, [0, 1, 0, 0, 0, 0, 0, 0])):
        dev_ctx.policy("float32", la.ptr, oa.ptr, aa.ptr, 1, 8, s.ptr, c.ptr, clip_low=low,
                       clip_high=HIGH, workspace=ws)
        dev_ctx.policy_grad("float32", g.ptr, la.ptr, oa.ptr, aa.ptr, 1, 8, c.ptr, clip_low=low,
                            clip_high=HIGH)
        dev_ctx.sync()
        assert c.get().tolist() == [8, 1, sum(cut)]
        assert ((g.get()[0] == 0) == (np.array(cut, bool) | (adv[0] == 0))).all()


@gpu
@pytest.mark.parametrize("dt", DTS)
def test_policy_far_references(dev_ctx, dt):
    """A reference that is -inf, the type's lowest value or merely far: the KL
    gradient is 1 - exp(q), to -1 and without a NaN."""
    low = {"float32": -3.4028234663852886e38, "bfloat16": -3.3895313892515355e38, "float16": -65504.0}[dt]
    ref = R.to_storage(np.array([[-np.inf, low, -60000.0, -30.0, -0.75, -0.5, 0.0, 0.75, 3.0]]), dt)
    zero = R.to_storage(np.zeros((1, 9)), dt)
    la, ra, aa, d = Arr(dev_ctx, zero), Arr(dev_ctx, ref), Arr(dev_ctx, np.zeros((1, 9), np.float32)), \
        Arr(dev_ctx, zero)
    c = Arr(dev_ctx, np.array([9, 1, 0], np.int64))
    dev_ctx.policy_grad(dt, d.ptr, la.ptr, la.ptr, aa.ptr, 1, 9, c.ptr, ref=ra.ptr, kl_coef=1.0)
    dev_ctx.sync()
    want = -np.expm1(R.from_storage(ref, dt)) / 9
    off = np.abs(R.from_storage(d.get(), dt) - want)
    # exp2 (2 u), its scaling (3 |q| u, |q| < 4 where the exponential is not nothing), the
    # difference (u), the weight's and the type's rounding
    assert (off <= (20 * U * np.maximum(1, np.exp(R.from_storage(ref, dt))) / 9 +
                    R.EPS[dt] * 1.01 * np.abs(want) + R.LEAST[dt])).all()


@gpu
def test_places_beyond_32_bits(dev_ctx):
    """More than 2^32 elements in a call, and row steps of more than 2^31: the
    far end gets what a call on it alone gets."""
    rows, cols = 65537, 65536 + 8
    n = rows * cols
    src, out = dev_ctx.alloc(2 * n), dev_ctx.alloc(2 * n)
    dev_ctx.fill("bfloat16", "round", 1, src, n)
    dev_ctx.sum_dropout("bfloat16", out.ptr, [src.ptr], rows, cols, 0.5, 3, offset=5)
    tail = dev_ctx.alloc(2 * 3 * cols)
    at = (rows - 3) * cols
    dev_ctx.sum_dropout("bfloat16", tail.ptr, [src.ptr + 2 * at], 3, cols, 0.5, 3, offset=5 + at)
    dev_ctx.sync()
    got = out.download(np.uint16, 3 * cols, 2 * at)
    assert (got == tail.download(np.uint16, 3 * cols)).all()
    keep = R.keep(3, 0, 5 + at, 3 * cols, 0.5)
    assert (got[~keep] == 0).all() and (got[keep] != 0).all()
    dev_ctx.sum_dropout_grad("bfloat16", out.ptr, src.ptr, rows, cols, 0.5, 3, offset=5)
    dev_ctx.sync()
    assert (out.download(np.uint16, 3 * cols, 2 * at) == got).all()
    # rows 2^31 + 64 elements apart, in the same memory
    ld, size = (1 << 31) + 64, 100
    assert 2 * ld + size <= n
    rng = np.random.default_rng(6)
    x = R.to_storage(rng.normal(size=(3, size)), "bfloat16")
    near, far = Arr(dev_ctx, x), Arr(dev_ctx, np.zeros_like(x))
    for r in range(2):
        src.upload(x[r], 2 * r * ld)
    c = [Arr(dev_ctx, np.zeros(size + 1, np.int64)) for _ in range(2)]
    s = [Arr(dev_ctx, np.zeros(size + 1, np.float32)) for _ in range(2)]
    i = Arr(dev_ctx, np.zeros((2, 1), np.int32))
    for k, (p, step) in enumerate(((near.ptr, 0), (src.ptr, ld))):
        dev_ctx.balance("bfloat16", p, i.ptr, 2, size, 1, c[k].ptr, s[k].ptr, index_dt="int32", ld=step)
    dev_ctx.balance_grad("bfloat16", out.ptr, src.ptr, 2, size, 1, c[0].ptr, balance_coef=1.0, ld=ld, ld_out=ld)
    dev_ctx.balance_grad("bfloat16", far.ptr, near.ptr, 2, size, 1, c[0].ptr, balance_coef=1.0)
    dev_ctx.sync()
    assert (c[0].get() == c[1].get()).all() and (s[0].get() == s[1].get()).all()
    for r in range(2):
        assert (out.download(np.uint16, size, 2 * r * ld) == far.get()[r]).all()
    adv = Arr(dev_ctx, np.ones(2, np.float32))
    pc, ps = Arr(dev_ctx, np.zeros(3, np.int64)), [Arr(dev_ctx, np.zeros(2, np.float32)) for _ in range(2)]
    ws = dev_ctx.alloc(dev_ctx.policy_workspace(2, size))
    for k, (p, step) in enumerate(((near.ptr, 0), (src.ptr, ld))):
        dev_ctx.policy("bfloat16", p, p, adv.ptr, 2, size, ps[k].ptr, pc.ptr, ref=p, adv_per_row=True, ld=step,
                       workspace=ws)
    dev_ctx.policy_grad("bfloat16", out.ptr, src.ptr, src.ptr, adv.ptr, 2, size, pc.ptr, adv_per_row=True, ld=ld)
    dev_ctx.policy_grad("bfloat16", far.ptr, near.ptr, near.ptr, adv.ptr, 2, size, pc.ptr, adv_per_row=True)
    dev_ctx.sync()
    assert (ps[0].get() == ps[1].get()).all() and pc.get().tolist() == [2 * size, 2, 0]
    for r in range(2):
        assert (out.download(np.uint16, size, 2 * r * ld) == far.get()[r]).all()
    for b in (src, out):
        b.free()


@gpu
def test_two_contexts_at_once(dev_ctx):
    """Two threads, a context, a stream and workspaces each: the results of one
    after the other."""
    import threading
    rng = np.random.default_rng(12)
    rows, cols = 3000, 257
    x = [rng.normal(size=(rows, cols)).astype(np.float32) for _ in range(2)]
    idx = [np.argsort(-v, 1)[:, :2].astype(np.int64) for v in x]

    def work(ctx, k, out):
        a, i = Arr(ctx, x[k]), Arr(ctx, idx[k])
        d, db = Arr(ctx, x[k] * 0), Arr(ctx, np.zeros(cols, np.float32))
        c, s = Arr(ctx, np.zeros(cols + 1, np.int64)), Arr(ctx, np.zeros(cols + 1, np.float32))
        loss, pc, ps = (Arr(ctx, np.zeros(n, t)) for n, t in ((3, np.float32), (3, np.int64), (2, np.float32)))
        ws = [ctx.alloc(max(16, n)) for n in (ctx.sum_dropout_grad_workspace(rows, cols),
                                              ctx.balance_workspace(rows, cols), ctx.policy_workspace(rows, cols))]
        for _ in range(20):
            ctx.sum_dropout_grad("float32", d.ptr, a.ptr, rows, cols, 0.1, k, dbias=db.ptr, workspace=ws[0])
            ctx.balance("float32", a.ptr, i.ptr, rows, cols, 2, c.ptr, s.ptr, loss=loss.ptr, balance_coef=1.0,
                        workspace=ws[1])
            ctx.policy("float32", a.ptr, d.ptr, a.ptr, rows, cols, ps.ptr, pc.ptr, workspace=ws[2])
        ctx.sync()
        out[k] = [v.get() for v in (d, db, c, s, loss, pc, ps)]
    alone, both = {}, {}
    for k in range(2):
        work(dev_ctx, k, alone)
    ctxs = [xucg_amd.DevContext(device=0) for _ in range(2)]
    ts = [threading.Thread(target=work, args=(ctxs[k], k, both)) for k in range(2)]
    for th in ts:
        th.start()
    for th in ts:
        th.join()
    for k in range(2):
        for v, w in zip(alone[k], both[k]):
            assert (v.view(np.uint8) == w.view(np.uint8)).all()
    for c in ctxs:
        c.close()


# ---- together ----------------------------------------------------------------------
@gpu
def test_a_step_of_four_members(dev_ctx):
    """Four members' shares of one step on one GPU: each member's rows of the
    combine with dropout are the whole's; statistics summed by the combine give
    the whole batch's losses, and the members' gradients are the whole's rows."""
    ctx, rng, world = dev_ctx, np.random.default_rng(11), 4
    rows, cols, e, k = 48, 64, 16, 2
    size = 2
    parts = [Arr(ctx, R.to_storage(rng.normal(size=(rows, cols)), "bfloat16")) for _ in range(world)]
    bias, res = (Arr(ctx, R.to_storage(rng.normal(size=s), "bfloat16")) for s in ((cols,), (rows, cols)))
    whole, cut = (Arr(ctx, np.zeros((rows, cols), np.uint16)) for _ in range(2))
    ctx.sum_dropout("bfloat16", whole.ptr, [q.ptr for q in parts], rows, cols, 0.1, 3, tag=1,
                    bias=bias.ptr, residual=res.ptr)

    class Peers:
        ptrs = [q.ptr for q in parts]
    for r in range(world):
        lo, _ = G.row_bounds(rows, world, r)
        at = lo * cols * size
        G.oneshot_reduce_scatter_dropout(ctx, Peers, cut.ptr + at, rows, cols, "bfloat16", 0.1, 3, r,
                                         world, tag=1, bias=bias.ptr, residual=res.ptr + at)
    ctx.sync()
    assert (whole.get() == cut.get()).all()

    # the router on the step's output: 32 bits, a share of padding
    x = rng.normal(size=(rows, e)).astype(np.float32)
    index = np.argsort(-x, 1)[:, :k].astype(np.int64)
    mask = (rng.random(rows) < 0.8).astype(np.uint8)
    xa, ia, ma = Arr(ctx, x), Arr(ctx, index), Arr(ctx, mask)
    stats = [(Arr(ctx, np.zeros(e + 1, np.int64)), Arr(ctx, np.zeros(e + 1, np.float32))) for _ in range(world)]
    ws = ctx.alloc(max(16, ctx.balance_workspace(rows, e)))
    loss = Arr(ctx, np.zeros(3, np.float32))
    bounds = [G.row_bounds(rows, world, r) for r in range(world)]
    for (lo, hi), (c, s) in zip(bounds, stats):
        ctx.balance("float32", xa.ptr + lo * e * 4, ia.ptr + lo * k * 8, hi - lo, e, k, c.ptr, s.ptr,
                    mask=ma.ptr + lo, workspace=ws)
    counts, sums = Arr(ctx, np.zeros(e + 1, np.int64)), Arr(ctx, np.zeros(e + 1, np.float32))
    assert ctx.reduce_multi("sum", "int64", counts.ptr, [c.ptr for c, _ in stats], 0, e + 1) == 0
    assert ctx.reduce_multi("sum", "float32", sums.ptr, [s.ptr for _, s in stats], 0, e + 1) == 0
    ctx.balance_loss(counts.ptr, sums.ptr, e, k, loss.ptr, balance_coef=0.01, z_coef=0.001)
    d_whole, d_cut = (Arr(ctx, np.zeros_like(x)) for _ in range(2))
    ctx.balance_grad("float32", d_whole.ptr, xa.ptr, rows, e, k, counts.ptr, mask=ma.ptr,
                     balance_coef=0.01, z_coef=0.001)
    for lo, hi in bounds:
        at = lo * e * 4
        ctx.balance_grad("float32", d_cut.ptr + at, xa.ptr + at, hi - lo, e, k, counts.ptr,
                         mask=ma.ptr + lo, balance_coef=0.01, z_coef=0.001)
    ctx.sync()
    wc, ws_ = check_balance(counts.get(), sums.get(), x.astype(np.float64), index, mask)
    rel, dl = balance_bounds(x.astype(np.float64), mask)
    want = R.balance_loss(wc, ws_, k, 0.01, 0.001)
    assert np.abs(loss.get() - want).max() <= (rel + 60 * U) * want[0] + 0.002 * dl * np.sqrt(ws_[e] / wc[e])
    assert (d_whole.get() == d_cut.get()).all()

    # answers shared out by rows; the mean of the group's sequences
    old = -rng.random((rows, 30)).astype(np.float32)
    lp = (old + rng.normal(size=old.shape) * 0.3).astype(np.float32)
    adv, m = rng.normal(size=rows).astype(np.float32), (rng.random(old.shape) < 0.7).astype(np.uint8)
    la, oa, aa, pm = (Arr(ctx, t) for t in (lp, old, adv, m))
    rt = Arr(ctx, np.zeros(rows, np.int32))
    ws = ctx.alloc(ctx.policy_workspace(rows, 30))
    stats = [(Arr(ctx, np.zeros(2, np.float32)), Arr(ctx, np.zeros(3, np.int64))) for _ in range(world)]
    kw = dict(adv_per_row=True, per_sequence=True)
    for (lo, hi), (s, c) in zip(bounds, stats):
        at = lo * 30
        ctx.policy("float32", la.ptr + at * 4, oa.ptr + at * 4, aa.ptr + lo * 4, hi - lo, 30, s.ptr, c.ptr,
                   mask=pm.ptr + at, row_tokens=rt.ptr + lo * 4, workspace=ws, **kw)
    sums, counts = Arr(ctx, np.zeros(2, np.float32)), Arr(ctx, np.zeros(3, np.int64))
    assert ctx.reduce_multi("sum", "float32", sums.ptr, [s.ptr for s, _ in stats], 0, 2) == 0
    assert ctx.reduce_multi("sum", "int64", counts.ptr, [c.ptr for _, c in stats], 0, 3) == 0
    ctx.policy_loss(sums.ptr, counts.ptr, loss.ptr, per_sequence=True)
    d = Arr(ctx, np.zeros_like(lp))
    for lo, hi in bounds:
        at = lo * 30
        ctx.policy_grad("float32", d.ptr + at * 4, la.ptr + at * 4, oa.ptr + at * 4, aa.ptr + lo * 4, hi - lo,
                        30, counts.ptr, mask=pm.ptr + at, row_tokens=rt.ptr + lo * 4, **kw)
    ctx.sync()
    l64, o64 = lp.astype(np.float64), old.astype(np.float64)
    a64 = np.broadcast_to(adv[:, None].astype(np.float64), lp.shape)
    pg, kl, was, dpg, dkl = R.policy_terms(l64, o64, a64, None, 0.2, 0.2)
    want, wc, tokens, sz = R.policy_stats(pg, kl, was, m, True)
    assert (counts.get() == wc).all() and (rt.get() == tokens).all()
    assert abs(loss.get()[0] - want[0] / wc[1]) <= 60 * U * sz[0] / wc[1]
    w = R.policy_grad(dpg, dkl, m, tokens, wc, True, 0.0)
    assert (np.abs(d.get() - w) <= 16 * U * np.abs(w) + 1e-30).all()


@gpu
@pytest.mark.parametrize("world", [2, 3])
def test_step_over_processes(world):
    """The group forms (group.py) over processes that share the GPU, their
    buffers mapped into one another."""
    from _launch import launch
    codes, outs = launch("_worker_step.py", world, timeout=200)
    assert codes == [0] * world, "\n".join(outs)


@gpu
def test_torch_tensors_and_captured_graphs(in_child):
    """Tensors are checked for type, place and strides; a captured step gives
    the eager step's bits at every replay, with other dropout state in each."""
    if in_child():
        return
    import torch
    ctx = xucg_amd.DevContext.on_torch_stream(0)
    rows, cols, e, k = 200, 520, 24, 2
    torch.manual_seed(0)

    def rand(*shape, dtype=torch.float32):
        return torch.randn(*shape, device="cuda").to(dtype)
    x, r, b = rand(rows, cols, dtype=torch.bfloat16), rand(rows, cols), rand(cols, dtype=torch.bfloat16)
    out, dsrc, dbias = torch.empty_like(r), torch.empty_like(x), torch.empty(cols, device="cuda")
    state = torch.tensor([5, 1], dtype=torch.int64, device="cuda")
    logits = rand(rows, e)
    index = torch.topk(logits, k).indices
    counts, sums = torch.empty(e + 1, dtype=torch.int64, device="cuda"), torch.empty(e + 1, device="cuda")
    loss, dlogits = torch.empty(3, device="cuda"), torch.empty_like(logits)
    lp, old = rand(rows, cols), rand(rows, cols)
    adv, mask = rand(rows), torch.rand(rows, cols, device="cuda") < 0.8
    ps, pc = torch.empty(2, device="cuda"), torch.empty(3, dtype=torch.int64, device="cuda")
    rt, dlp = torch.empty(rows, dtype=torch.int32, device="cuda"), torch.empty_like(lp)
    ws = [torch.empty(max(16, n), dtype=torch.uint8, device="cuda")
          for n in (ctx.sum_dropout_grad_workspace(rows, cols), ctx.balance_workspace(rows, e),
                    ctx.policy_workspace(rows, cols))]

    def step():
        ctx.sum_dropout("bfloat16", out, [x, x], rows, cols, 0.2, 0, bias=b, residual=r,
                        out_dt="float32", rng=state)
        ctx.sum_dropout_grad("bfloat16", dsrc, out, rows, cols, 0.2, 0, dbias=dbias,
                             grad_dt="float32", workspace=ws[0], rng=state)
        ctx.balance("float32", logits, index, rows, e, k, counts, sums, loss=loss, balance_coef=1.0,
                    workspace=ws[1])
        ctx.balance_grad("float32", dlogits, logits, rows, e, k, counts, balance_coef=1.0)
        ctx.policy("float32", lp, old, adv, rows, cols, ps, pc, mask=mask, row_tokens=rt,
                   adv_per_row=True, per_sequence=True, workspace=ws[2])
        ctx.policy_grad("float32", dlp, lp, old, adv, rows, cols, pc, mask=mask, row_tokens=rt,
                        adv_per_row=True, per_sequence=True)
        return [t.clone() for t in (out, dsrc, dbias, counts, sums, loss, dlogits, ps, pc, rt, dlp)]
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=ctx.torch_stream):
        held = step()
    for n in range(4):
        state.copy_(torch.tensor([5 + n, 1 << n]))
        logits.copy_(torch.randn_like(logits))
        index.copy_(torch.topk(logits, k).indices)
        lp.copy_(torch.randn_like(lp))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        want = step()
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert torch.equal(g, w), n
    # refusals
    for what, call in (
            ("srcs", lambda: ctx.sum_dropout("bfloat16", out, [r], rows, cols, 0.1, 1, out_dt="float32")),
            ("dst", lambda: ctx.sum_dropout("bfloat16", out.cpu(), [x], rows, cols, 0.1, 1, out_dt="float32")),
            ("dst", lambda: ctx.sum_dropout("float32", r.t(), [r], rows, cols, 0.1, 1)),
            ("residual", lambda: ctx.sum_dropout("float32", out, [r], rows, cols, 0.1, 1, residual=r[1:])),
            ("rng", lambda: ctx.sum_dropout("float32", out, [r], rows, cols, 0.1, 1, rng=state[:1])),
            ("index", lambda: ctx.balance("float32", logits, index.int(), rows, e, k, counts, sums, workspace=ws[1])),
            ("counts", lambda: ctx.balance("float32", logits, index, rows, e, k, counts[:-1], sums, workspace=ws[1])),
            ("logits", lambda: ctx.balance("float32", logits, index, rows, e, k, counts, sums, ld=e + 1,
                                           workspace=ws[1])),
            ("adv", lambda: ctx.policy("float32", lp, old, adv, rows, cols, ps, pc, workspace=ws[2])),
            ("workspace", lambda: ctx.policy("float32", lp, old, adv, rows, cols, ps, pc, adv_per_row=True,
                                             workspace=ws[2].cpu()))):
        with pytest.raises(ValueError, match=what):
            call()
    with pytest.raises(xucg_amd.UcsError, match="workspace"):
        ctx.policy("float32", lp, old, adv, rows, cols, ps, pc, adv_per_row=True, workspace=ws[2][:-1])
    # a slice with a wider step
    wide = torch.randn(rows, e + 9, device="cuda")
    ctx.balance("float32", wide[:, :e], index, rows, e, k, counts, sums, ld=e + 9, workspace=ws[1])
    got = sums.clone()
    ctx.balance("float32", wide[:, :e].contiguous(), index, rows, e, k, counts, sums, workspace=ws[1])
    torch.cuda.synchronize()
    assert torch.equal(got, sums)
    ctx.close()
