"""One rank of the training-step test: every rank lives on cuda:0, maps the
others' buffers, takes its rows of the combine with dropout, and sums the
router's and the policy's statistics with the one-shot allreduce. Each rank
holds the whole's inputs and checks its share against them."""
import os
import sys

import numpy as np
import torch.distributed as dist

import xucg_amd
from oracle import train_ref as R
from xucg_amd import group as G

U = 2.0 ** -24


def main():
    rank, world = int(os.environ["RANK"]), int(os.environ["WORLD_SIZE"])
    dist.init_process_group("gloo", rank=rank, world_size=world)
    ctx = xucg_amd.DevContext(device=0)

    def barrier():
        ctx.sync()
        dist.barrier()

    def check(ok, what):
        if not ok:
            print(f"rank {rank}: MISMATCH {what}", flush=True)
            sys.exit(1)

    rng = np.random.default_rng(2)                # the same on every rank
    rows, cols, p = 101, 96, 0.2
    parts = [R.to_storage(rng.normal(size=(rows, cols)), "bfloat16") for _ in range(world)]
    bias = R.to_storage(rng.normal(size=cols), "bfloat16")
    res = rng.normal(size=(rows, cols)).astype(np.float32)
    mine, b, r, out = (ctx.alloc(x.nbytes) for x in (parts[0], bias, res, res))
    lo, hi = G.row_bounds(rows, world, rank)
    mine.upload(parts[rank])
    b.upload(bias)
    r.upload(res[lo:hi])
    peers = G.PeerBuffers(ctx, mine.ptr, rank, world, dist)
    barrier()
    got_lo, got_hi = G.oneshot_reduce_scatter_dropout(
        ctx, peers, out.ptr, rows, cols, "bfloat16", p, 17, rank, world, tag=4, offset=40,
        bias=b.ptr, residual=r.ptr, out_dt="float32")
    barrier()
    check((got_lo, got_hi) == (lo, hi), "rows")
    keep = R.keep(17, 4, 40, rows * cols, p).reshape(rows, cols)[lo:hi]
    want, size = R.sum_dropout([R.from_storage(q, "bfloat16")[lo:hi] for q in parts],
                               R.from_storage(bias, "bfloat16"), res[lo:hi].astype(np.float64), keep, p)
    got = out.download(np.float32, (hi - lo) * cols).reshape(hi - lo, cols)
    # world - 1 sums, bias, scale and its rounding, residual, the last one
    check((np.abs(got - want) <= (world + 5) * U * size * 1.01).all(), "reduce-scatter with dropout")
    peers.close()

    # an allreduce of the framework's own: send and receive buffers mapped once
    send, recv = ctx.alloc(4096), ctx.alloc(4096)
    sp = G.PeerBuffers(ctx, send.ptr, rank, world, dist)
    rp = G.PeerBuffers(ctx, recv.ptr, rank, world, dist)

    def allreduce(buf, dt, count):
        n = count * {"int64": 8, "float32": 4}[dt]
        ctx.copy_multi([send.ptr], [buf.ptr], n)
        barrier()
        G.oneshot_allreduce(ctx, sp, rp, count, dt, "sum", rank, world, barrier)
        ctx.copy_multi([buf.ptr], [recv.ptr], n)
        barrier()

    e, k = 24, 3
    x = rng.normal(size=(rows, e)).astype(np.float32)
    index = np.argsort(-x, 1)[:, :k].astype(np.int32)
    mask = (rng.random(rows) < 0.7).astype(np.uint8)
    xa, ia, ma, d = (ctx.alloc(t.nbytes) for t in (x, index, mask, x))
    xa.upload(x[lo:hi])
    ia.upload(index[lo:hi])
    ma.upload(mask[lo:hi])
    counts, sums, loss = ctx.alloc(8 * (e + 1)), ctx.alloc(4 * (e + 1)), ctx.alloc(16)
    ws = ctx.alloc(max(16, ctx.balance_workspace(rows, e)))
    G.group_balance(ctx, allreduce, "float32", xa.ptr, ia.ptr, hi - lo, e, k, counts, sums, loss.ptr,
                    mask=ma.ptr, balance_coef=0.5, z_coef=0.1, index_dt="int32", workspace=ws)
    ctx.balance_grad("float32", d.ptr, xa.ptr, hi - lo, e, k, counts.ptr, mask=ma.ptr,
                     balance_coef=0.5, z_coef=0.1)
    ctx.sync()
    wc, wsum = R.balance_stats(x.astype(np.float64), index, mask)
    check((counts.download(np.int64, e + 1) == wc).all(), "counts")
    want = R.balance_loss(wc, wsum, k, 0.5, 0.1)
    # logits within 8 of one another, 24 terms, 101 tokens: test_train_ops' bounds
    tol = (6 * 8 + e + 10 + rows + 20) * U
    check((np.abs(loss.download(np.float32, 3) - want) <= 3 * tol * np.abs(want).max()).all(), "balance loss")
    g = R.balance_grad(x.astype(np.float64), mask, wc, k, 0.5, 0.1)
    got = d.download(np.float32, (hi - lo) * e).reshape(hi - lo, e)
    check((np.abs(got - g[lo:hi]) <= 8 * tol * np.abs(g).max()).all(), "balance gradient")

    old = -rng.random((rows, 50)).astype(np.float32)
    lp = (old + rng.normal(size=old.shape) * 0.3).astype(np.float32)
    ref = (old + rng.normal(size=old.shape) * 0.3).astype(np.float32)
    adv = rng.normal(size=old.shape).astype(np.float32)
    m = (rng.random(old.shape) < 0.6).astype(np.uint8)
    m[5] = 0
    la, oa, ra, aa, pm, dl = (ctx.alloc(t.nbytes) for t in (lp, old, ref, adv, m, lp))
    for buf, t in ((la, lp), (oa, old), (ra, ref), (aa, adv), (pm, m)):
        buf.upload(t[lo:hi])
    ps, pc, rt = ctx.alloc(16), ctx.alloc(32), ctx.alloc(4 * rows)
    ws = ctx.alloc(ctx.policy_workspace(rows, 50))
    for seq in (False, True):
        G.group_policy(ctx, allreduce, "float32", la.ptr, oa.ptr, aa.ptr, hi - lo, 50, ps, pc, loss.ptr,
                       ref=ra.ptr, mask=pm.ptr, row_tokens=rt.ptr, per_sequence=seq, kl_coef=0.2,
                       workspace=ws)
        ctx.policy_grad("float32", dl.ptr, la.ptr, oa.ptr, aa.ptr, hi - lo, 50, pc.ptr, ref=ra.ptr,
                        mask=pm.ptr, row_tokens=rt.ptr, per_sequence=seq, kl_coef=0.2)
        ctx.sync()
        pg, kl, cut, dpg, dkl = R.policy_terms(*(t.astype(np.float64) for t in (lp, old, adv, ref)), 0.2, 0.2)
        s, c, tokens, size = R.policy_stats(pg, kl, cut, m, seq)
        check((pc.download(np.int64, 3) == c).all(), "policy counts")
        want = R.policy_loss(s, c, seq, 0.2)
        n = c[1] if seq else c[0]
        check(np.abs(loss.download(np.float32, 3) - want).max() <= 100 * U * size.sum() / n, "policy loss")
        g = R.policy_grad(dpg, dkl, m, tokens, c, seq, 0.2)
        got = dl.download(np.float32, (hi - lo) * 50).reshape(hi - lo, 50)
        check((np.abs(got - g[lo:hi]) <= 80 * U * np.abs(g).max()).all(), "policy gradient")
    sp.close()
    rp.close()
    dist.barrier()
    ctx.close()
    dist.destroy_process_group()
    print(f"rank {rank}: ok", flush=True)


if __name__ == "__main__":
    main()
