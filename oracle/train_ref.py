"""The training-step operators in 64-bit numpy, from their definitions
(include/ucg_builtin_dev.h): what the tests hold the kernels to."""
import numpy as np

EPS = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}   # half a step
LEAST = {"float32": 2.0 ** -149, "bfloat16": 2.0 ** -133, "float16": 2.0 ** -24}
STORAGE = {"float32": np.float32, "bfloat16": np.uint16, "float16": np.float16}


def to_storage(x, dt):
    """x rounded to dt, in its storage type (bfloat16: the upper 16 bits)."""
    if dt != "bfloat16":
        return np.asarray(x, np.float64).astype(np.float32).astype(STORAGE[dt])
    b = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    r = (b + 0x7fff + ((b >> 16) & 1)) >> 16
    return np.where(np.isnan(x), 0x7fc0, r).astype(np.uint16)


def from_storage(x, dt):
    if dt != "bfloat16":
        return x.astype(np.float64)
    return (x.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


# ---- dropout -------------------------------------------------------------------
def philox(counter, key, rounds=10):
    """Philox-4x32 (Salmon et al., SC 2011): counter [4, n], key [2] -> [4, n]."""
    c = [np.asarray(x, np.uint64) for x in counter]
    k = [int(key[0]), int(key[1])]
    low, s32 = np.uint64(0xffffffff), np.uint64(32)
    for _ in range(rounds):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> s32) ^ c[1] ^ np.uint64(k[0]), b & low,
             (a >> s32) ^ c[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & 0xffffffff, (k[1] + 0xBB67AE85) & 0xffffffff]
    return np.stack(c)


def threshold(p):
    return int(np.rint(p * 65536))


def scale(p):
    t = threshold(p)
    return 65536 / (65536 - t) if t < 65536 else 0.0


def keep(seed, tag, offset, n, p):
    g = np.arange(offset, offset + n, dtype=np.uint64)
    group, lane = g >> np.uint64(3), (g & np.uint64(7)).astype(np.int64)
    full = np.zeros_like(group)
    w = philox([group & np.uint64(0xffffffff), group >> np.uint64(32), full + np.uint64(tag & 0xffffffff),
                full + np.uint64(tag >> 32)], (seed & 0xffffffff, seed >> 32))
    half = (w[lane >> 1, np.arange(n)] >> (16 * (lane & 1)).astype(np.uint64)) & np.uint64(0xffff)
    return half >= threshold(p)


def sum_dropout(srcs, bias, residual, mask, p):
    """(value, what its rounding errors are relative to)"""
    x, size = sum(srcs), sum(np.abs(s) for s in srcs)
    if bias is not None:
        x, size = x + bias, size + np.abs(bias)
    out, size = np.where(mask, x * scale(p), 0.0), np.where(mask, size * scale(p), 0.0)
    if residual is not None:
        out, size = out + residual, size + np.abs(residual)
    return out, size


# ---- balance loss --------------------------------------------------------------
def softmax(x):
    """probabilities and log sum exp by rows; a row of -inf alone has neither"""
    top = x.max(1, initial=-np.inf, keepdims=True)
    top = np.where(np.isneginf(top), 0.0, top)
    w = np.exp(x - top)
    s = w.sum(1, keepdims=True)
    with np.errstate(divide="ignore", invalid="ignore"):
        p = np.where(s > 0, w / s, 0.0)
        lse = np.where(s > 0, np.log(s) + top, 0.0)
    return p, lse[:, 0]


def balance_stats(x, index, mask):
    """counts [E + 1], sums [E + 1]"""
    e = x.shape[1]
    live = np.ones(len(x), bool) if mask is None else mask != 0
    p, lse = softmax(x[live])
    named = index[live].reshape(-1)
    named = named[(named >= 0) & (named < e)]
    counts = np.append(np.bincount(named, minlength=e), live.sum()).astype(np.int64)
    return counts, np.append(p.sum(0), (lse ** 2).sum())


def balance_loss(counts, sums, topk, coef, z_coef):
    e, n = len(counts) - 1, float(counts[-1])
    if n == 0:
        return np.zeros(3)
    b = coef * e / (topk * n * n) * (counts[:e].astype(np.float64) @ sums[:e])
    z = z_coef * sums[e] / n if z_coef else 0.0
    return np.array([b + z, b, z])


def balance_grad(x, mask, counts, topk, coef, z_coef, g=1.0):
    e, n = x.shape[1], float(counts[-1])
    live = np.ones(len(x), bool) if mask is None else mask != 0
    d = np.zeros_like(x)
    if n:
        p, lse = softmax(x[live])
        c = counts[:e].astype(np.float64)
        d[live] = g * (coef * e / (topk * n * n) * p * (c - (p @ c)[:, None]) +
                       2 * z_coef / n * lse[:, None] * p)
    return d


# ---- policy loss ---------------------------------------------------------------
def policy_terms(logp, old, adv, ref, low, high):
    """pg, kl, cut, dpg, dkl of every token; `cut` goes by the 32-bit difference"""
    d32 = (logp.astype(np.float32) - old.astype(np.float32))
    up, down = np.float32(np.log1p(high)), np.float32(np.log1p(-low) if low < 1 else -np.inf)
    cut = ((adv > 0) & (d32 > up)) | ((adv < 0) & (d32 < down))
    r = np.exp(logp - old)
    pg = -adv * np.where(cut, np.where(adv > 0, 1 + high, 1 - low), r)
    q = np.zeros_like(logp) if ref is None else ref - logp
    return pg, np.expm1(q) - q, cut, np.where(cut, 0.0, -adv * r), -np.expm1(q)


def policy_stats(pg, kl, cut, mask, per_sequence):
    """sums [2], counts [3], row_tokens, and the sums of the terms' sizes"""
    live = mask != 0
    rows = live.sum(1)
    w = 1.0 / np.maximum(rows, 1) if per_sequence else np.ones(len(rows))
    pg, kl = np.where(live, pg, 0.0), np.where(live, kl, 0.0)
    sums = np.array([(pg.sum(1) * w).sum(), (kl.sum(1) * w).sum()])
    size = np.array([(np.abs(pg).sum(1) * w).sum(), (np.abs(kl).sum(1) * w).sum()])
    return sums, np.array([rows.sum(), (rows > 0).sum(), (live & cut).sum()]), rows, size


def policy_loss(sums, counts, per_sequence, kl_coef):
    n = counts[1] if per_sequence else counts[0]
    pg, kl = (sums[0] / n, sums[1] / n) if n else (0.0, 0.0)
    return np.array([pg + kl_coef * kl, pg, kl])


def policy_grad(dpg, dkl, mask, rows, counts, per_sequence, kl_coef, g=1.0):
    n = counts[1] if per_sequence else counts[0]
    w = np.full(len(rows), g / n if n else 0.0)
    if per_sequence:
        w = w / np.maximum(rows, 1)
    return np.where(mask != 0, (dpg + kl_coef * dkl) * w[:, None], 0.0)
