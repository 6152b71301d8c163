"""Python handle over the C-ABI device combine (include/ucg_builtin_dev.h).

`DevContext` is the per-group device context of UCG's builtin planner
(`struct ucg_builtin_group_ctx`, reference builtin/builtin.c:66-90). Its
methods map one-to-one onto the C entry points; buffers are passed as raw
device pointers (ints), `DevBuffer` objects, or torch tensors (`data_ptr()`).
Torch is not required by this module.
"""
import ctypes

import numpy as np

from . import _lib
from ._lib import check, dt_index, op_index, dist_index, DTYPE_SIZE

NP_STORAGE = {"int8": np.int8, "uint8": np.uint8, "int16": np.int16,
              "uint16": np.uint16, "int32": np.int32, "uint32": np.uint32,
              "int64": np.int64, "uint64": np.uint64, "float16": np.float16,
              "bfloat16": np.uint16, "float32": np.float32,
              "float64": np.float64}


def _ptr(x):
    if x is None:
        return None
    if isinstance(x, int):
        return x
    if isinstance(x, (DevBuffer, HostBuffer)):
        return x.ptr
    if hasattr(x, "data_ptr"):
        return x.data_ptr()
    if isinstance(x, np.ndarray):
        return x.ctypes.data
    raise TypeError(f"cannot take a device pointer of {type(x)}")


_DT = {name: i for i, name in enumerate(_lib.DTYPES)}


_TORCH = {}     # name -> torch dtype, filled by the tensors that come (torch not imported)


def _is_dtype(dtype, name):
    """whether a torch dtype is the type `name` (a uint8 mask may be bool)"""
    known = str(dtype).rpartition(".")[2]
    if known == name:
        _TORCH[name] = dtype
    return known == name or (name == "uint8" and known == "bool")


def _name(dt):
    return dt if isinstance(dt, str) else _lib.DTYPES[dt]


def dtype_size(dt):
    return DTYPE_SIZE[dt_index(dt)]


def is_supported(dt, op):
    return bool(_lib.dev().ucg_builtin_dev_is_supported(dt_index(dt), op_index(op)))


def device_count():
    return _lib.dev().ucg_builtin_dev_device_count()


class DevBuffer:
    """A device buffer owned by a DevContext: hipMalloc'ed, or (shareable)
    HIP virtual memory that peers map by its physical allocation."""

    def __init__(self, ctx, nbytes, shareable=False):
        self.ctx = ctx
        self.nbytes = nbytes
        fn = (_lib.dev().ucg_builtin_dev_malloc_shareable if shareable
              else _lib.dev().ucg_builtin_dev_malloc)
        self.ptr = fn(ctx.handle, nbytes)
        if not self.ptr:
            raise MemoryError(f"device allocation of {nbytes} B failed: {_lib.last_error()}")

    def offset(self, nbytes):
        return self.ptr + nbytes

    def upload(self, arr, offset=0):
        arr = np.ascontiguousarray(arr)
        assert offset + arr.nbytes <= self.nbytes
        check(_lib.dev().ucg_builtin_dev_memcpy(self.ctx.handle, self.ptr + offset,
                                                arr.ctypes.data, arr.nbytes), "memcpy H2D")

    def download(self, dtype, count, offset=0):
        out = np.empty(count, dtype=dtype)
        assert offset + out.nbytes <= self.nbytes
        check(_lib.dev().ucg_builtin_dev_memcpy(self.ctx.handle, out.ctypes.data,
                                                self.ptr + offset, out.nbytes), "memcpy D2H")
        return out

    def free(self):
        if self.ptr:
            _lib.dev().ucg_builtin_dev_free(self.ctx.handle, self.ptr)
            self.ptr = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


class HostBuffer:
    """Pinned (hipHostMalloc) host memory viewed as a numpy array."""

    def __init__(self, nbytes):
        self.nbytes = nbytes
        self.ptr = _lib.dev().ucg_builtin_dev_host_alloc(nbytes)
        if not self.ptr:
            raise MemoryError(f"hipHostMalloc({nbytes}) failed: {_lib.last_error()}")

    def view(self, dtype, count=None):
        dtype = np.dtype(dtype)
        count = self.nbytes // dtype.itemsize if count is None else count
        buf = (ctypes.c_char * (count * dtype.itemsize)).from_address(self.ptr)
        return np.frombuffer(buf, dtype=dtype, count=count)

    def free(self):
        if self.ptr:
            _lib.dev().ucg_builtin_dev_host_free(self.ptr)
            self.ptr = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


class DevContext:
    """Per-group device context: one HIP stream, a pinned staging ring and the
    per-step device accumulator."""

    def __init__(self, device=-1, stream=None, stage_bytes=0, stage_slots=0,
                 zcopy_bytes=0, completion="signal"):
        if stream is not None and stream == 0:
            # the C ABI reads NULL as "create a stream": the legacy null stream
            # cannot be shared, and a private non-blocking stream would not be
            # ordered with the caller's work. Share a real stream instead.
            raise ValueError("stream 0 (the null stream) cannot be shared; use "
                             "DevContext.on_torch_stream()")
        L = _lib.dev()
        # zcopy_bytes: 0 = the library default (64 KiB), None = never
        zc = _lib.ZCOPY_NEVER if zcopy_bytes is None else zcopy_bytes
        # completion: how stage_end waits ("signal": pinned completion word,
        # "sync": hipStreamSynchronize)
        p = _lib.DevCtxParams(device, stream, stage_bytes, stage_slots, zc,
                              _lib.COMPLETION[completion])
        h = ctypes.c_void_p()
        check(L.ucg_builtin_dev_ctx_create(ctypes.byref(p), ctypes.byref(h)),
              "ucg_builtin_dev_ctx_create")
        self.handle = h.value
        self.device = L.ucg_builtin_dev_ctx_device(h)

    @classmethod
    def on_torch_stream(cls, device=0, **kw):
        """A context that launches on torch's current stream, made a fresh
        (non-null) stream here: torch ops, RCCL collectives (which order
        themselves against the caller's current stream) and this context's
        combines are then stream-ordered with no host syncs."""
        import torch
        torch.cuda.set_device(device)
        s = torch.cuda.Stream(device=device)
        torch.cuda.set_stream(s)
        ctx = cls(device=device, stream=s.cuda_stream, **kw)
        ctx.torch_stream = s        # keep the stream alive with the context
        return ctx

    # -- lifecycle --------------------------------------------------------
    def close(self):
        if getattr(self, "handle", None):
            _lib.dev().ucg_builtin_dev_ctx_destroy(self.handle)
            self.handle = None

    def __enter__(self):
        return self

    def __exit__(self, *a):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    @property
    def stream(self):
        return _lib.dev().ucg_builtin_dev_ctx_stream(self.handle)

    def sync(self):
        check(_lib.dev().ucg_builtin_dev_sync(self.handle), "ucg_builtin_dev_sync")

    # -- memory -----------------------------------------------------------
    def alloc(self, nbytes, shareable=False):
        return DevBuffer(self, nbytes, shareable)

    def debug_ptr(self, ptr):
        """what the runtime and the shim know about a device address, and the
        process's recent memory events near it (diagnostics)"""
        buf = ctypes.create_string_buffer(1 << 16)
        _lib.dev().ucg_builtin_dev_debug_ptr(self.handle, _ptr(ptr), buf, len(buf))
        return buf.value.decode(errors="replace")

    def fill(self, dt, dist, seed, buf, count):
        check(_lib.dev().ucg_builtin_dev_fill(self.handle, dt_index(dt), dist_index(dist),
                                              seed, _ptr(buf), count), "ucg_builtin_dev_fill")

    # -- combine ----------------------------------------------------------
    def reduce(self, op, dt, dst, src, count):
        """dst[i] = src[i] (op) dst[i] on device pointers (async)."""
        return _lib.dev().ucg_builtin_dev_reduce(self.handle, op_index(op), dt_index(dt),
                                                 _ptr(dst), _ptr(src), count)

    def reduce_checked(self, op, dt, dst, src, count):
        check(self.reduce(op, dt, dst, src, count), "ucg_builtin_dev_reduce")

    def reduce_multi(self, op, dt, dst, srcs, self_index, count):
        arr = (ctypes.c_void_p * len(srcs))(*[_ptr(s) for s in srcs])
        return _lib.dev().ucg_builtin_dev_reduce_multi(self.handle, op_index(op),
                                                       dt_index(dt), _ptr(dst), arr,
                                                       len(srcs), self_index, count)

    def reduce_tree(self, op, dt, dst, srcs, count):
        """Tree fan-in: acc = srcs[0]; acc = srcs[m] (op) acc for m = 1.. ."""
        arr = (ctypes.c_void_p * len(srcs))(*[_ptr(s) for s in srcs])
        return _lib.dev().ucg_builtin_dev_reduce_tree(self.handle, op_index(op),
                                                      dt_index(dt), _ptr(dst), arr,
                                                      len(srcs), count)

    def gather_multi(self, dst, srcs, shard_bytes):
        """dst[r * shard_bytes:...] = srcs[r][:shard_bytes] in one launch."""
        arr = (ctypes.c_void_p * len(srcs))(*[_ptr(s) for s in srcs])
        return _lib.dev().ucg_builtin_dev_gather_multi(self.handle, _ptr(dst), arr,
                                                       len(srcs), shard_bytes)

    def copy_multi(self, dsts, srcs, nbytes):
        """dsts[i][:nbytes] = srcs[i][:nbytes] for every pair, one launch."""
        n = len(dsts)
        if len(srcs) != n:
            raise ValueError("copy_multi: as many sources as destinations")
        da = (ctypes.c_void_p * n)(*[_ptr(d) for d in dsts])
        sa = (ctypes.c_void_p * n)(*[_ptr(s) for s in srcs])
        return _lib.dev().ucg_builtin_dev_copy_multi(self.handle, da, sa, n, nbytes)

    # -- operators of a training step beside the combine -------------------
    def _at(self, name, x, dt, n, row=0, step=0):
        """The address of operand `name`. A torch tensor is held to what the
        call reads or writes there: the type, this context's device, n
        elements without gaps - or in rows of `row` that lie `step` apart."""
        if x is None or x.__class__ is int:
            return x
        try:
            dtype, address = x.dtype, x.data_ptr()
        except AttributeError:
            if not isinstance(x, (DevBuffer, HostBuffer)):
                raise TypeError(f"{name}: device memory wanted, got {type(x)}") from None
            if not x.ptr:             # NULL is an operand left out
                raise ValueError(f"{name}: the buffer is freed")
            span = n if step == row or not n else (n // row - 1) * step + row
            if span * DTYPE_SIZE[_DT[dt]] > x.nbytes:
                raise ValueError(f"{name}: a buffer of {span} {dt} wanted, got {x.nbytes} bytes")
            return x.ptr
        if (step == row and x.is_contiguous() and x.numel() == n and
                dtype is _TORCH.get(dt) and x.get_device() == self.device):
            return address
        if not _is_dtype(dtype, dt):
            raise ValueError(f"{name}: {dt} wanted, got {dtype}")
        if x.get_device() != self.device:
            raise ValueError(f"{name}: a tensor on cuda:{self.device} wanted, got {x.device}")
        if x.numel() != n:
            raise ValueError(f"{name}: {n} elements wanted, got {tuple(x.shape)}")
        if step == row:
            if not x.is_contiguous():
                raise ValueError(f"{name}: a contiguous tensor wanted, got strides {x.stride()}")
        elif n and (x.dim() != 2 or x.shape[1] != row or (row > 1 and x.stride(1) != 1) or
                    (n > row and x.stride(0) != step)):
            raise ValueError(f"{name}: rows of {row}, {step} apart, wanted, got "
                             f"{tuple(x.shape)} with strides {x.stride()}")
        return address

    def sum_dropout(self, dt, dst, srcs, rows, cols, p, seed, tag=0, offset=0, bias=None,
                    residual=None, out_dt=None, rng=None):
        """dst = residual + dropout(sum of srcs + bias), the mask a function of
        (seed, tag, offset + element) that is never stored
        (ucg_builtin_dev_sum_dropout). rng: device memory holding {seed, tag}."""
        dt, at, n = _name(dt), self._at, rows * cols
        out_dt = dt if out_dt is None else _name(out_dt)
        srcs = [at("srcs", s, dt, n) for s in srcs]
        q = _lib.DropoutParams(_DT[dt], _DT[out_dt], rows, cols, p, seed, tag, offset,
                               at("rng", rng, "int64", 2) or 0)
        st = _lib.dev().ucg_builtin_dev_sum_dropout(
            self.handle, q, at("dst", dst, out_dt, n), _lib.addresses(srcs), len(srcs),
            at("bias", bias, dt, cols), at("residual", residual, out_dt, n))
        if st:
            check(st, "ucg_builtin_dev_sum_dropout")

    @staticmethod
    def sum_dropout_grad_workspace(rows, cols):
        """bytes of sum_dropout_grad's workspace (with dbias)"""
        return _lib.dev().ucg_builtin_dev_sum_dropout_grad_workspace(rows, cols)

    def sum_dropout_grad(self, dt, dsrc, grad, rows, cols, p, seed, tag=0, offset=0, dbias=None,
                         grad_dt=None, workspace=None, rng=None):
        """dsrc = the gradient of every source of sum_dropout, dbias (cols
        floats) = the bias' (ucg_builtin_dev_sum_dropout_grad)."""
        dt, at, n = _name(dt), self._at, rows * cols
        grad_dt = dt if grad_dt is None else _name(grad_dt)
        q = _lib.DropoutParams(_DT[dt], _DT[grad_dt], rows, cols, p, seed, tag, offset,
                               at("rng", rng, "int64", 2) or 0)
        ws, nbytes = self._workspace(workspace, self.sum_dropout_grad_workspace, rows, cols)
        st = _lib.dev().ucg_builtin_dev_sum_dropout_grad(
            self.handle, q, at("dsrc", dsrc, dt, n), at("grad", grad, grad_dt, n),
            at("dbias", dbias, "float32", cols), ws, nbytes)
        if st:
            check(st, "ucg_builtin_dev_sum_dropout_grad")

    def _workspace(self, workspace, need, *sizes):
        """A workspace's address and bytes. An address alone is taken to hold
        what the call needs, as the C caller says it does."""
        if workspace is None:
            return None, 0
        if isinstance(workspace, int):
            return workspace, need(*sizes)
        if hasattr(workspace, "data_ptr"):
            if workspace.get_device() != self.device or not workspace.is_contiguous():
                raise ValueError(f"workspace: a contiguous tensor on cuda:{self.device} wanted")
            return workspace.data_ptr(), workspace.nbytes
        if not isinstance(workspace, (DevBuffer, HostBuffer)):
            raise TypeError(f"workspace: device memory wanted, got {type(workspace)}")
        if not workspace.ptr:
            raise ValueError("workspace: the buffer is freed")
        return workspace.ptr, workspace.nbytes

    @staticmethod
    def balance_workspace(tokens, experts):
        """bytes of balance's workspace"""
        return _lib.dev().ucg_builtin_dev_balance_workspace(tokens, experts)

    def balance(self, dt, logits, index, tokens, experts, topk, counts, sums, mask=None,
                loss=None, balance_coef=0.0, z_coef=0.0, index_dt="int64", ld=0, ld_index=0,
                workspace=None):
        """counts (experts + 1 int64: uses of each expert, tokens) and sums
        (experts + 1 float32: probability of each expert, squared log sum exp)
        of this member's tokens: what the group adds up
        (ucg_builtin_dev_balance). loss: 3 floats, for a group of one."""
        dt, index_dt, at = _name(dt), _name(index_dt), self._at
        q = _lib.BalanceParams(_DT[dt], _DT[index_dt], tokens, experts, topk, ld, ld_index, 0,
                               balance_coef, z_coef)
        ws, nbytes = self._workspace(workspace, self.balance_workspace, tokens, experts)
        st = _lib.dev().ucg_builtin_dev_balance(
            self.handle, q,
            at("logits", logits, dt, tokens * experts, experts, ld or experts),
            at("index", index, index_dt, tokens * topk, topk, ld_index or topk),
            at("mask", mask, "uint8", tokens), at("counts", counts, "int64", experts + 1),
            at("sums", sums, "float32", experts + 1), at("loss", loss, "float32", 3), ws, nbytes)
        if st:
            check(st, "ucg_builtin_dev_balance")

    def balance_loss(self, counts, sums, experts, topk, loss, balance_coef=0.0, z_coef=0.0):
        """loss (3 floats: whole, balance part, z part) from the group's counts
        and sums (ucg_builtin_dev_balance_loss)."""
        at = self._at
        q = _lib.BalanceParams(_DT["float32"], _DT["int64"], 0, experts, topk, 0, 0, 0,
                               balance_coef, z_coef)
        check(_lib.dev().ucg_builtin_dev_balance_loss(
            self.handle, q, at("counts", counts, "int64", experts + 1),
            at("sums", sums, "float32", experts + 1), at("loss", loss, "float32", 3)),
            "ucg_builtin_dev_balance_loss")

    def balance_grad(self, dt, dlogits, logits, tokens, experts, topk, counts, mask=None,
                     base=None, grad_loss=None, balance_coef=0.0, z_coef=0.0, ld=0, ld_out=0):
        """dlogits = base + grad_loss * the loss' gradient, with the group's
        counts (ucg_builtin_dev_balance_grad)."""
        dt, at, n = _name(dt), self._at, tokens * experts
        q = _lib.BalanceParams(_DT[dt], _DT["int64"], tokens, experts, topk, ld, 0, ld_out,
                               balance_coef, z_coef)
        st = _lib.dev().ucg_builtin_dev_balance_grad(
            self.handle, q, at("logits", logits, dt, n, experts, ld or experts),
            at("mask", mask, "uint8", tokens), at("counts", counts, "int64", experts + 1),
            at("base", base, dt, n, experts, ld_out or experts),
            at("grad_loss", grad_loss, "float32", 1),
            at("dlogits", dlogits, dt, n, experts, ld_out or experts))
        if st:
            check(st, "ucg_builtin_dev_balance_grad")

    @staticmethod
    def policy_workspace(rows, cols):
        """bytes of policy's workspace"""
        return _lib.dev().ucg_builtin_dev_policy_workspace(rows, cols)

    def policy(self, dt, logp, old, adv, rows, cols, sums, counts, ref=None, mask=None,
               row_tokens=None, adv_per_row=False, per_sequence=False, clip_low=0.2,
               clip_high=0.2, kl_coef=0.0, loss=None, ld=0, workspace=None):
        """sums (2 float32: clipped policy term, KL) and counts (3 int64:
        tokens, rows that have one, cut tokens) of this member's answers: what
        the group adds up (ucg_builtin_dev_policy). loss: 3 floats, for a group
        of one."""
        dt, at, n, step = _name(dt), self._at, rows * cols, ld or cols
        q = _lib.PolicyParams(_DT[dt], adv_per_row, per_sequence, rows, cols, ld, clip_low,
                              clip_high, kl_coef)
        ws, nbytes = self._workspace(workspace, self.policy_workspace, rows, cols)
        st = _lib.dev().ucg_builtin_dev_policy(
            self.handle, q, at("logp", logp, dt, n, cols, step), at("old", old, dt, n, cols, step),
            at("ref", ref, dt, n, cols, step),
            at("adv", adv, "float32", rows) if adv_per_row else
            at("adv", adv, "float32", n, cols, step),
            at("mask", mask, "uint8", n, cols, step), at("sums", sums, "float32", 2),
            at("counts", counts, "int64", 3), at("row_tokens", row_tokens, "int32", rows),
            at("loss", loss, "float32", 3), ws, nbytes)
        if st:
            check(st, "ucg_builtin_dev_policy")

    def policy_loss(self, sums, counts, loss, per_sequence=False, kl_coef=0.0):
        """loss (3 floats: whole, policy mean, KL mean) from the group's sums
        and counts (ucg_builtin_dev_policy_loss)."""
        at = self._at
        q = _lib.PolicyParams(_DT["float32"], 0, per_sequence, 0, 0, 0, 0.0, 0.0, kl_coef)
        check(_lib.dev().ucg_builtin_dev_policy_loss(
            self.handle, q, at("sums", sums, "float32", 2), at("counts", counts, "int64", 3),
            at("loss", loss, "float32", 3)), "ucg_builtin_dev_policy_loss")

    def policy_grad(self, dt, dlogp, logp, old, adv, rows, cols, counts, ref=None, mask=None,
                    row_tokens=None, adv_per_row=False, per_sequence=False, clip_low=0.2,
                    clip_high=0.2, kl_coef=0.0, grad_loss=None, ld=0):
        """dlogp = grad_loss * the loss' gradient, with the group's counts
        (ucg_builtin_dev_policy_grad)."""
        dt, at, n, step = _name(dt), self._at, rows * cols, ld or cols
        q = _lib.PolicyParams(_DT[dt], adv_per_row, per_sequence, rows, cols, ld, clip_low,
                              clip_high, kl_coef)
        st = _lib.dev().ucg_builtin_dev_policy_grad(
            self.handle, q, at("logp", logp, dt, n, cols, step), at("old", old, dt, n, cols, step),
            at("ref", ref, dt, n, cols, step),
            at("adv", adv, "float32", rows) if adv_per_row else
            at("adv", adv, "float32", n, cols, step),
            at("mask", mask, "uint8", n, cols, step),
            at("row_tokens", row_tokens, "int32", rows), at("counts", counts, "int64", 3),
            at("grad_loss", grad_loss, "float32", 1), at("dlogp", dlogp, dt, n, cols, step))
        if st:
            check(st, "ucg_builtin_dev_policy_grad")

    def combine_host(self, op, dt, dst_host, src_host, count):
        return _lib.dev().ucg_builtin_dev_combine_host(self.handle, op_index(op),
                                                       dt_index(dt), _ptr(dst_host),
                                                       _ptr(src_host), count)

    def stage_begin(self, host_dst, nbytes):
        return _lib.dev().ucg_builtin_dev_stage_begin(self.handle, _ptr(host_dst), nbytes)

    def combine(self, op, dt, dst_offset, host_src, count):
        return _lib.dev().ucg_builtin_dev_combine(self.handle, op_index(op), dt_index(dt),
                                                  dst_offset, _ptr(host_src), count)

    def stage_end(self):
        return _lib.dev().ucg_builtin_dev_stage_end(self.handle)

    # -- peer mapping -----------------------------------------------------
    def ipc_export(self, buf):
        """Opaque bytes naming `buf` for another process (xGMI peer)."""
        h = (ctypes.c_char * _lib.IPC_HANDLE_BYTES)()
        check(_lib.dev().ucg_builtin_dev_ipc_export(self.handle, _ptr(buf), h),
              "ucg_builtin_dev_ipc_export")
        return bytes(h)

    def ipc_import(self, blob):
        """Map a peer buffer exported by ipc_export(); returns a device pointer."""
        h = (ctypes.c_char * _lib.IPC_HANDLE_BYTES).from_buffer_copy(blob)
        p = ctypes.c_void_p()
        check(_lib.dev().ucg_builtin_dev_ipc_import(self.handle, h, ctypes.byref(p)),
              "ucg_builtin_dev_ipc_import")
        return p.value

    def ipc_release(self, ptr):
        check(_lib.dev().ucg_builtin_dev_ipc_release(self.handle, ptr),
              "ucg_builtin_dev_ipc_release")

    # -- profiling --------------------------------------------------------
    def profile_reduce(self, op, dt, dst, src, count, iters):
        us = ctypes.c_double()
        check(_lib.dev().ucg_builtin_dev_profile_reduce(self.handle, op_index(op),
                                                        dt_index(dt), _ptr(dst), _ptr(src),
                                                        count, iters, ctypes.byref(us)),
              "ucg_builtin_dev_profile_reduce")
        return us.value

    def profile_reduce_multi(self, op, dt, dst, srcs, self_index, count, iters):
        """reduce_multi launched `iters` times back to back between two HIP
        events on the context stream: average us per launch."""
        us = ctypes.c_double()
        arr = (ctypes.c_void_p * len(srcs))(*[_ptr(s) for s in srcs])
        check(_lib.dev().ucg_builtin_dev_profile_reduce_multi(
                  self.handle, op_index(op), dt_index(dt), _ptr(dst), arr, len(srcs),
                  self_index, count, iters, ctypes.byref(us)),
              "ucg_builtin_dev_profile_reduce_multi")
        return us.value

    def profile_stream(self, kind, dst, src, nbytes, iters):
        """Measured ceiling in the combine's geometry: kind 0 reads both
        buffers (no stores), kind 1 copies src -> dst. Average us per launch."""
        us = ctypes.c_double()
        check(_lib.dev().ucg_builtin_dev_profile_stream(self.handle, kind, _ptr(dst), _ptr(src),
                                                        nbytes, iters, ctypes.byref(us)),
              "ucg_builtin_dev_profile_stream")
        return us.value

    def counters(self):
        out = (ctypes.c_uint64 * _lib.NCOUNTERS)()
        _lib.dev().ucg_builtin_dev_counters(self.handle, out)
        c = {"launches": out[0], "combined_bytes": out[1], "h2d_bytes": out[2],
             "d2h_bytes": out[3], "zcopy_bytes": out[4], "signal_waits": out[5]}
        # the process-wide accounting beside the context's own (retired
        # address ranges and their cap: ucg_builtin_dev_mem_stats)
        c.update(_lib.mem_stats())
        return c


def use_shareable_torch_memory():
    """Route torch's device allocations through the shim's shareable
    allocator (torch.cuda.memory.CUDAPluggableAllocator over
    ucg_builtin_dev_torch_alloc / _free), so that every tensor of this process
    can be exported by its physical allocation (ucg_builtin_dev_ipc_export).
    Must run before torch allocates any device memory in the process; it
    replaces torch's caching allocator (every allocation is a VMM mapping of
    whole 2 MiB granules, every free waits for the device)."""
    import torch
    _lib.dev()                       # built, and loaded after torch's HIP runtime
    alloc = torch.cuda.memory.CUDAPluggableAllocator(
        _lib.DEV_LIB, "ucg_builtin_dev_torch_alloc", "ucg_builtin_dev_torch_free")
    torch.cuda.memory.change_current_allocator(alloc)
