"""The training-step operators where their kernels go further than a small case
takes them: members without work, loops past their first pass, in-place
gradients, many rows to a lane, values at the ends of their range. The oracle
and the arrays are test_train_ops.py's; every bound is counted from the
operations that a value goes through (u = 2^-24 for each in fp32)."""
import numpy as np
import pytest

import test_train_ops as near
import xucg_amd
from oracle import train_ref as R
from test_train_ops import DTS, U, Arr, balance_bounds, gpu, ptr
from xucg_amd import group as G


# ---- refusals (CPU) --------------------------------------------------------------------
def test_freed_buffers_are_refused():
    """A buffer that was freed has the address NULL, which for an operand that may
    be left out would mean that: the call would run without bias or mask."""
    ctx = xucg_amd.DevContext.__new__(xucg_amd.DevContext)   # no GPU is needed to refuse
    ctx.handle, ctx.device = None, 0
    for kind in (xucg_amd.DevBuffer, xucg_amd.HostBuffer):
        gone = kind.__new__(kind)
        gone.ptr, gone.nbytes = None, 1 << 20
        at = [k << 20 for k in range(1, 9)]
        for what, call in (
                ("bias", lambda: ctx.sum_dropout("float32", at[0], at[1:2], 4, 8, 0.1, 1, bias=gone)),
                ("residual", lambda: ctx.sum_dropout("float32", at[0], at[1:2], 4, 8, 0.1, 1, residual=gone)),
                ("rng", lambda: ctx.sum_dropout("float32", at[0], at[1:2], 4, 8, 0.1, 1, rng=gone)),
                ("dbias", lambda: ctx.sum_dropout_grad("float32", at[0], at[1], 4, 8, 0.1, 1, dbias=gone)),
                ("mask", lambda: ctx.balance("float32", at[0], at[1], 4, 8, 2, at[2], at[3], mask=gone)),
                ("base", lambda: ctx.balance_grad("float32", at[0], at[1], 4, 8, 2, at[2], base=gone)),
                ("ref", lambda: ctx.policy("float32", *at[:3], 4, 8, *at[3:5], ref=gone, workspace=at[5])),
                ("grad_loss", lambda: ctx.policy_grad("float32", *at[:4], 4, 8, at[4], grad_loss=gone)),
                ("workspace", lambda: ctx.policy("float32", *at[:3], 4, 8, *at[3:5], workspace=gone))):
            with pytest.raises(ValueError, match=f"{what}: the buffer is freed"):
                call()
    for what in (np.zeros(64, np.uint8), "ws"):
        with pytest.raises(TypeError, match="workspace: device memory wanted"):
            ctx.policy("float32", *at[:3], 4, 8, *at[3:5], workspace=what)


# ---- members without work ------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("cols", [0, 5, 16385, 20000, 1 << 20, (1 << 31) - 1])
def test_policy_of_a_member_without_rows(dev_ctx, dt, cols):
    """No rows of any length: zeros, also where a row would be many parts; in a
    group, the member adds its zeros and takes part in the allreduce."""
    s, c = Arr(dev_ctx, np.ones(2, np.float32)), Arr(dev_ctx, np.ones(3, np.int64))
    loss, ws = Arr(dev_ctx, np.ones(3, np.float32)), dev_ctx.alloc(dev_ctx.policy_workspace(0, cols))
    for per_row in (False, True):
        for ref in (None, 1 << 20):           # never looked at
            dev_ctx.policy(dt, None, None, None, 0, cols, s.ptr, c.ptr, ref=ref, adv_per_row=per_row,
                           per_sequence=per_row, loss=loss.ptr, workspace=ws)
            dev_ctx.policy_grad(dt, None, None, None, None, 0, cols, c.ptr, ref=ref, adv_per_row=per_row)
            dev_ctx.sync()
            assert not s.get().any() and not c.get().any() and not loss.get().any()
            for a in (s, c, loss):
                a.buf.upload(a.whole)         # ones again
    other = {"float32": Arr(dev_ctx, np.array([6, 3], np.float32)), "int64": Arr(dev_ctx, np.array([4, 2, 1], np.int64))}
    joined = []

    def allreduce(buf, t, n):
        """the other member's share is added"""
        joined.append(t)
        assert dev_ctx.reduce("sum", t, buf, other[t].ptr, n) == 0
    G.group_policy(dev_ctx, allreduce, dt, None, None, None, 0, cols, s.ptr, c.ptr, loss.ptr, kl_coef=0.5,
                   workspace=ws)
    dev_ctx.sync()
    assert sorted(joined) == ["float32", "int64"]
    assert c.get().tolist() == [4, 2, 1] and loss.get().tolist() == [1.875, 1.5, 0.75]


# ---- the balance gradient's centre ---------------------------------------------------
@gpu
@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("experts,topk,dropped", [(64, 8, 0.5), (60, 8, 0.9), (512, 4, 0.3), (1000, 2, 0.97)])
def test_balance_grad_of_dropped_choices(dev_ctx, dt, experts, topk, dropped):
    """Counts that are near one another and far below tokens * topk / experts:
    choices with an index outside the experts are counted nowhere. The
    gradient's p (c - p.c) needs the counts' differences alone, so its bound
    goes by their spread: each term of the dot has the spread, the error of a
    probability and one rounding for itself and each of its sums."""
    rng = np.random.default_rng(experts)
    tokens, members = 40, 1 << 16
    x = R.from_storage(R.to_storage(rng.normal(size=(tokens, experts)), dt), dt)
    mean = int(members * topk * (1 - dropped) / experts)
    counts = np.append(mean + rng.integers(-3, 4, experts), members).astype(np.int64)
    la, ca, d = Arr(dev_ctx, R.to_storage(x, dt)), Arr(dev_ctx, counts), Arr(dev_ctx, R.to_storage(np.zeros_like(x), dt))
    coef = float(members) ** 2 / experts        # the result is of the counts' own size
    dev_ctx.balance_grad(dt, d.ptr, la.ptr, tokens, experts, topk, ca.ptr, balance_coef=coef)
    dev_ctx.sync()
    want = R.balance_grad(x, None, counts, topk, coef, 0.0)
    rel, _ = balance_bounds(x, None)
    p, _ = R.softmax(x)
    # differences of two counts: 6 at most
    size = 8 * coef * experts / topk / float(members) ** 2
    tol = p * size * (2 * rel + (experts + 8) * U)
    off = np.abs(R.from_storage(d.get(), dt) - want)
    tol = tol + R.EPS[dt] * (np.abs(want) + tol) * 1.01 + R.LEAST[dt]
    assert (off <= tol).all(), (off / tol).max()



# ---- many rows to a lane -------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dt,rows,cols,offset", [
    ("float32", 1 << 21, 8, 0), ("float32", 1 << 21, 8, 3), ("float32", 1 << 18, 65, 1),
    ("bfloat16", 1 << 20, 16, 0), ("bfloat16", 300, (1 << 19) + 8, 0), ("bfloat16", 300, (1 << 19) + 3, 0)])
def test_bias_gradient_of_many_rows(dev_ctx, dt, rows, cols, offset):
    """Columns that begin with ones and go on with values that a sum of 1 in 32
    bits loses whole. At most 32 rows are added up in 32 bits, a part and the
    result are rounded once more: 33 u of the sum of sizes."""
    head = min(rows // 64, 1 << 15)
    one, small = R.to_storage(np.array([1.0, 2.0 ** -24]), dt)
    g = np.full((rows, cols), small)
    g[:head] = one
    ga, d = Arr(dev_ctx, g), Arr(dev_ctx, np.zeros_like(g))
    db = Arr(dev_ctx, np.ones(cols, np.float32))
    ws = dev_ctx.alloc(max(16, dev_ctx.sum_dropout_grad_workspace(rows, cols)))
    dev_ctx.sum_dropout_grad(dt, d.ptr, ga.ptr, rows, cols, 0.0, 1, offset=offset, dbias=db.ptr, workspace=ws)
    dev_ctx.sync()
    want = head + (rows - head) * 2.0 ** -24
    assert np.abs(db.get() - want).max() <= 33 * U * want
    assert (d.get() == g).all()


@gpu
@pytest.mark.parametrize("dt,experts", [("bfloat16", 512), ("float16", 256), ("float32", 256), ("bfloat16", 60)])
def test_balance_sums_of_many_rows(dev_ctx, dt, experts):
    """Blocks that begin with rows whose probability for expert 0 is 1, and
    whose log sum exp is 16, and go on with rows of which a sum in 32 bits would
    lose both values whole. At most 32 rows are added up in 32 bits, then six
    steps over lanes, one over waves, a part's and the last rounding: 41 u. A
    probability of 1 is exact, of 1 - 2^-24 to 2 u; the others weigh nothing."""
    tokens = (1 << 27) // max(experts, 64)           # 64 rows and more to a lane
    low, z = 16.7, 0.0035                            # exp(-low) = 0.94 * 2^-24, z^2 = 0.8 * 256 * 2^-24
    kinds = np.full((2, experts), -np.inf)
    kinds[0, 0], kinds[1, 0], kinds[1, 1] = 16.0, z - low, z
    kinds = R.to_storage(kinds, dt)
    head = np.arange(tokens) % (tokens // 256) < 16 * 64 // min(64, max(1, experts * 2 // 16))
    p, lse = R.softmax(R.from_storage(kinds, dt))
    la = Arr(dev_ctx, kinds[np.where(head, 0, 1)])
    ia = Arr(dev_ctx, np.zeros((tokens, 1), np.int32))
    c, s = Arr(dev_ctx, np.zeros(experts + 1, np.int64)), Arr(dev_ctx, np.zeros(experts + 1, np.float32))
    ws = dev_ctx.alloc(max(16, dev_ctx.balance_workspace(tokens, experts)))
    dev_ctx.balance(dt, la.ptr, ia.ptr, tokens, experts, 1, c.ptr, s.ptr, index_dt="int32", workspace=ws)
    dev_ctx.sync()
    n = np.array([head.sum(), (~head).sum()], np.float64)
    got = s.get().astype(np.float64)
    want = np.append(n @ p, n @ lse ** 2)
    assert (np.abs(got - want) <= 43 * U * want).all()
    assert c.get()[0] == tokens == c.get()[-1]


# ---- values at the ends of their range -----------------------------------------------
@gpu
@pytest.mark.parametrize("per_row", [False, True])
def test_policy_without_advantage(dev_ctx, per_row):
    """A = 0 (of either sign) gives 0 for any ratio, also one that is infinite
    in 32 bits, and cuts nothing; a NaN stays one."""
    d = np.array([0.5, 87, 89, 200, 1e30, np.inf, -5, -200, -np.inf, 88.72, 1, 2, 3], np.float32)
    for sign in (0.0, -0.0):
        la, oa = Arr(dev_ctx, d[None]), Arr(dev_ctx, np.zeros((1, len(d)), np.float32))
        aa = Arr(dev_ctx, np.full(1 if per_row else (1, len(d)), sign, np.float32))
        s, c, g = Arr(dev_ctx, np.ones(2, np.float32)), Arr(dev_ctx, np.ones(3, np.int64)), Arr(dev_ctx, d[None])
        ws = dev_ctx.alloc(dev_ctx.policy_workspace(1, len(d)))

        def run():
            dev_ctx.policy("float32", la.ptr, oa.ptr, aa.ptr, 1, len(d), s.ptr, c.ptr, adv_per_row=per_row,
                           workspace=ws)
            dev_ctx.policy_grad("float32", g.ptr, la.ptr, oa.ptr, aa.ptr, 1, len(d), c.ptr, adv_per_row=per_row)
            dev_ctx.sync()
        run()
        assert s.get().tolist() == [0, 0] and c.get().tolist() == [len(d), 1, 0]
        assert (g.get() == 0).all()
        x = d[None].copy()
        x[0, 3] = np.nan
        la = Arr(dev_ctx, x)
        run()
        assert np.isnan(s.get()[0]) and (np.isnan(g.get()[0]) == np.isnan(x[0])).all()


@gpu
def test_policy_ratio_is_as_near_as_documented(dev_ctx):
    """The gradient of A = -1 over one token is the ratio itself (clip_low = 1
    cuts none): off by (1.25 |d| + 2) u, for d = 0 not at all."""
    d = np.append(np.linspace(-80, 80, 4001), [0.0, 1e-30, 88.0, -87.0]).astype(np.float32)[None]
    la, oa = Arr(dev_ctx, d), Arr(dev_ctx, d * 0)
    aa, g, c = Arr(dev_ctx, -np.ones(1, np.float32)), Arr(dev_ctx, d * 0), Arr(dev_ctx, np.ones(3, np.int64))
    dev_ctx.policy_grad("float32", g.ptr, la.ptr, oa.ptr, aa.ptr, 1, d.size, c.ptr, adv_per_row=True, clip_low=1.0)
    dev_ctx.sync()
    d64 = d.astype(np.float64)
    off = np.abs(g.get() / np.exp(d64) - 1) / U
    assert (off <= 1.25 * np.abs(d64) + 2).all()
    assert (g.get()[d == 0] == 1).all()


# ---- loops past their first pass -----------------------------------------------------
# The sizes are the smallest that make each kernel's loops repeat: the rows of
# the bias' gradient (256 parts of 4 lanes, four rows a pass: 4096), the rows of
# the balance gradient (1024 blocks), the rows and the parts of the policy join
# (64 blocks; 8 parts to each of 64 lanes), the parts of the policy kernels.
@gpu
@pytest.mark.parametrize("dt,grad_dt", [("float32", "float32"), ("bfloat16", "bfloat16"),
                                        ("float16", "float16"), ("bfloat16", "float32"),
                                        ("float16", "float32")])
@pytest.mark.parametrize("rows,cols,offset", [(4101, 512, 0), (4101, 515, 5)])
def test_bias_gradient_of_several_passes(dev_ctx, dt, grad_dt, rows, cols, offset):
    near.test_sum_dropout_grad(dev_ctx, dt, grad_dt, rows, cols, offset)


@gpu
@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("tokens,experts,topk", [(5000, 1000, 4), (17000, 256, 8)])
def test_balance_of_several_passes(dev_ctx, dt, tokens, experts, topk):
    near.test_balance(dev_ctx, dt, tokens, experts, topk)


@gpu
@pytest.mark.parametrize("dt,rows,cols", [(dt, *s) for dt in DTS for s in ((20000, 5), (1, 600000))] +
                         [("float32", 1, 5000001), ("bfloat16", 2, 4300005)])
def test_policy_of_several_passes(dev_ctx, dt, rows, cols):
    near.test_policy(dev_ctx, dt, rows, cols)


@gpu
def test_policy_of_very_many_rows(dev_ctx):
    """More rows than a grid has at once (2^20 blocks of 256), one token each, all
    of ratio 1: the sums are the advantages', whole numbers."""
    rows = (1 << 28) + 300
    adv = np.ones(rows, np.float32)
    adv[-300:] = 3
    want = -(1 << 28) - 900.0
    x, a = dev_ctx.alloc(2 * rows), dev_ctx.alloc(4 * rows)
    a.upload(adv)
    chunk = np.zeros(1 << 26, np.uint16)
    for at in range(0, 2 * rows, chunk.nbytes):
        x.upload(chunk[:(2 * rows - at) // 2], at)
    d, ws = dev_ctx.alloc(2 * rows), dev_ctx.alloc(dev_ctx.policy_workspace(rows, 1))
    s, c = Arr(dev_ctx, np.ones(2, np.float32)), Arr(dev_ctx, np.ones(3, np.int64))
    kw = dict(adv_per_row=True)
    dev_ctx.policy("bfloat16", x, x, a, rows, 1, s.ptr, c.ptr, workspace=ws, **kw)
    dev_ctx.policy_grad("bfloat16", d, x, x, a, rows, 1, c.ptr, **kw)
    dev_ctx.sync()
    assert s.get().tolist() == [np.float32(want), 0] and c.get().tolist() == [rows, rows, 0]
    got = d.download(np.uint16, rows)
    one, three = R.to_storage(np.array([-1.0, -3.0]) / rows, "bfloat16")
    assert (got[:1 << 28] == one).all() and (got[1 << 28:] == three).all()
    for b in (x, a, d, ws):
        b.free()


# ---- gradients in place --------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("rows,cols,offset", [(5, 13, 3), (4101, 512, 8), (4101, 515, 5), (1 << 18, 65, 1)])
def test_dropout_gradient_in_place(dev_ctx, dt, rows, cols, offset):
    """dsrc = grad: the bits of the call that is not in place."""
    rng = np.random.default_rng(cols)
    g = R.to_storage(rng.normal(size=(rows, cols)).astype(np.float32), dt)
    for with_bias in (True, False):
        got = []
        for in_place in (False, True):
            ga, db = Arr(dev_ctx, g), Arr(dev_ctx, np.ones(cols, np.float32))
            d = ga if in_place else Arr(dev_ctx, g * 0)
            ws = dev_ctx.alloc(max(16, dev_ctx.sum_dropout_grad_workspace(rows, cols)))
            dev_ctx.sum_dropout_grad(dt, d.ptr, ga.ptr, rows, cols, 0.3, 7, offset=offset,
                                     dbias=db.ptr if with_bias else None, workspace=ws)
            dev_ctx.sync()
            got.append((d.get(), db.get()))
        assert (got[0][0] == got[1][0]).all() and (got[0][1] == got[1][1]).all()


@gpu
@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("tokens,experts", [(9, 5), (5000, 1000), (17000, 256), (70000, 8), (30011, 60)])
def test_balance_gradient_in_place(dev_ctx, dt, tokens, experts):
    """dlogits = logits and dlogits = base, also while the next rows are on the
    way: the bits of the call that is not in place."""
    rng = np.random.default_rng(tokens)
    x, base = (R.to_storage(rng.normal(size=(tokens, experts)).astype(np.float32) * s, dt) for s in (2, 1e-3))
    mask = (rng.random(tokens) < 0.8).astype(np.uint8)
    counts = np.append(rng.integers(0, tokens, experts), max(1, mask.sum())).astype(np.int64)
    ca, ma = Arr(dev_ctx, counts), Arr(dev_ctx, mask)
    got = {}
    for where in ("apart", "logits", "base", "apart, no base", "logits, no base"):
        la, ba = Arr(dev_ctx, x), Arr(dev_ctx, base)
        d = {"l": la, "b": ba}.get(where[0]) or Arr(dev_ctx, x * 0)
        dev_ctx.balance_grad(dt, d.ptr, la.ptr, tokens, experts, 2, ca.ptr, mask=ma.ptr, balance_coef=0.5,
                             z_coef=0.1, base=None if "no base" in where else ba.ptr)
        dev_ctx.sync()
        got[where] = d.get()
        assert where[0] == "l" or (la.get() == x).all()
        assert where[0] == "b" or (ba.get() == base).all()
    assert (got["logits"] == got["apart"]).all() and (got["base"] == got["apart"]).all()
    assert (got["logits, no base"] == got["apart, no base"]).all()


@gpu
@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("rows,cols", [(3, 7), (300, 33), (20000, 5), (9, 4100), (1, 600000)])
def test_policy_gradient_in_place(dev_ctx, dt, rows, cols):
    """dlogp = logp, old or ref: the bits of the call that is not in place."""
    rng = np.random.default_rng(cols)
    old = -rng.random((rows, cols)).astype(np.float32) * 3
    arrays = [R.to_storage(a, dt) for a in (old + rng.normal(size=old.shape).astype(np.float32) * 0.3, old,
                                            old + rng.normal(size=old.shape).astype(np.float32) * 0.3)]
    adv = Arr(dev_ctx, rng.normal(size=old.shape).astype(np.float32))
    mask = (rng.random(old.shape) < 0.7).astype(np.uint8)
    ma, ca = Arr(dev_ctx, mask), Arr(dev_ctx, np.array([mask.sum() + 1, rows, 0], np.int64))
    got = {}
    for where in (None, 0, 1, 2):
        a = [Arr(dev_ctx, v) for v in arrays]
        d = Arr(dev_ctx, arrays[0] * 0) if where is None else a[where]
        dev_ctx.policy_grad(dt, d.ptr, a[0].ptr, a[1].ptr, adv.ptr, rows, cols, ca.ptr, ref=a[2].ptr, mask=ma.ptr,
                            kl_coef=0.3)
        dev_ctx.sync()
        got[where] = d.get()
        for i in range(3):
            assert i == where or (a[i].get() == arrays[i]).all()
    assert all((got[w] == got[None]).all() for w in got)


# ---- sums near their bound -----------------------------------------------------------
def sums_tolerance(x, mask, ws):
    """What the balance sums may be off: a probability's and a log sum exp's own
    error, 32 rows of a lane, six steps over lanes, one over waves, a part's and
    the last rounding - whatever the number of tokens."""
    rel, dl = balance_bounds(x, mask)
    e, n = x.shape[1], len(x) if mask is None else int((mask != 0).sum())
    z = 2 * dl * np.sqrt(n * ws[e]) + n * dl * dl
    return np.append((rel + 41 * U) * ws[:e], z + 41 * U * ws[e])


@gpu
@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("tokens,experts,topk", [(40000, 8, 2), (33000, 5, 1), (20000, 16, 2)])
def test_balance_sums_miss_no_token(dev_ctx, dt, tokens, experts, topk):
    """The bound is tight enough to see a token of tens of thousands: without
    any one of some, the oracle's own sums are past it."""
    rng = np.random.default_rng(experts)
    x, index, mask = near.balance_inputs(rng, dt, tokens, experts, topk, np.int64, "some")
    _, _, c, s, _ = near.run_balance(dev_ctx, dt, x, index, mask)
    wc, ws = R.balance_stats(x, index, mask)
    tol = sums_tolerance(x, mask, ws)
    assert (c.get() == wc).all()
    off = np.abs(s.get().astype(np.float64) - ws)
    assert (off <= tol).all(), (off / tol).max()
    p, lse = R.softmax(x)
    for t in np.flatnonzero(mask)[:50]:
        assert (np.append(p[t], lse[t] ** 2) > 2 * tol).any()
