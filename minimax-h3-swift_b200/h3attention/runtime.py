"""Per-device handle on the C ABI: one ``h3c_ctx`` per CUDA device.

Torch tensors are accepted for convenience; only their device pointers,
shapes and strides cross the boundary.
"""
from __future__ import annotations

import ctypes as C
import threading
from typing import Dict, Optional

from . import _lib


def _stream_ptr(stream) -> Optional[int]:
    import torch

    s = stream if stream is not None else torch.cuda.current_stream()
    return s.cuda_stream or None


def view_of(t, layout: str) -> _lib.View:
    """h3c_view of a bf16 tensor.  layout "SHD": [S, H, 128]; "HSD": [H, S, 128]."""
    if t.stride(-1) != 1:
        raise ValueError("head_dim must be contiguous")
    if layout == "SHD":
        tok, head = t.stride(0), t.stride(1)
    elif layout == "HSD":
        head, tok = t.stride(0), t.stride(1)
    else:
        raise ValueError(layout)
    return _lib.View(t.data_ptr(), tok, head)


def _bview(name, t, layout: str, device: int, shape=None):
    """``(h3c_bview, (batch, tokens, heads))`` of a bf16 tensor on ``device``:
    [B, S, H, 128] or [S, H, 128] ("SHD"), [B, H, S, 128] or [H, S, 128]
    ("HSD").  ``shape``: the (batch, tokens, heads) it must have."""
    import torch

    if t.dtype is not torch.bfloat16 or t.device.type != "cuda" or t.device.index != device:
        raise ValueError(f"{name} must be bfloat16 on cuda:{device}, got {t.dtype} on {t.device}")
    size, stride = t.shape, t.stride()
    if len(size) == 3:
        size, stride = (1, *size), (0, *stride)
    if len(size) != 4:
        raise ValueError(f"{name} must have 3 or 4 axes, got {tuple(t.shape)}")
    if layout == "SHD":
        b, s, h, d = size
        view = _lib.BView(t.data_ptr(), stride[0], stride[1], stride[2])
    elif layout == "HSD":
        b, h, s, d = size
        view = _lib.BView(t.data_ptr(), stride[0], stride[2], stride[1])
    else:
        raise ValueError(layout)
    if stride[3] != 1 and d > 1:
        raise ValueError(f"{name}: head_dim must be contiguous")
    if d != 128:
        raise _lib.H3CError(_lib.H3C_ERR_UNSUPPORTED, f"{name}: head_dim must be 128, got {d}")
    if shape is not None and (b, s, h) != shape:
        raise ValueError(f"{name} must have {shape} (batch, tokens, heads), got {(b, s, h)}")
    return view, (b, s, h)


def _vector(name, t, dtype, shape, device: int) -> int:
    """Device pointer of a contiguous tensor of the given type and shape."""
    if t.dtype is not dtype or t.device.type != "cuda" or t.device.index != device or tuple(t.shape) != shape \
            or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {shape} on cuda:{device}, got "
                         f"{t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


class Runtime:
    _lock = threading.Lock()
    _by_device: Dict[int, "Runtime"] = {}

    def __init__(self, device: int):
        self.L = _lib.load()
        self.device = device
        h = C.c_void_p()
        _lib.check(self.L.h3c_init(device, C.byref(h)), what=f"h3c_init(device={device})")
        self.ctx = h

    @classmethod
    def get(cls, device: Optional[int] = None) -> "Runtime":
        if device is None:
            import torch

            device = torch.cuda.current_device()
        with cls._lock:
            rt = cls._by_device.get(device)
            if rt is None:
                rt = cls._by_device[device] = Runtime(device)
            return rt

    @staticmethod
    def device_count() -> int:
        n = C.c_int(0)
        _lib.load().h3c_device_count(C.byref(n))
        return n.value

    def _check(self, st: int):
        _lib.check(st, self.ctx)

    def device_info(self) -> dict:
        info = _lib.DevInfo()
        self._check(self.L.h3c_device_info(self.ctx, C.byref(info)))
        d = {f: getattr(info, f) for f, _ in _lib.DevInfo._fields_}
        d["name"] = info.name.decode()
        d["pci_bus_id"] = info.pci_bus_id.decode()
        return d

    # ------------------------------------------------------------ attention
    def attn_args(self, q, k, v, out, layout, scale, blocks, flags=0, heads=None, head_offset=0,
                  head_count=None, q_norm=None, k_norm=None, eps=1e-6, rope_table=None):
        seq_axis = 0 if layout == "SHD" else 1
        head_axis = 1 - seq_axis
        H = q.shape[head_axis] if heads is None else heads
        a = _lib.AttnArgs()
        a.q, a.k, a.v, a.out = (view_of(t, layout) for t in (q, k, v, out))
        a.seq_len = q.shape[seq_axis]
        a.heads = H
        a.head_dim = q.shape[-1]
        a.head_offset = head_offset
        a.head_count = H - head_offset if head_count is None else head_count
        a.scale = scale
        rp, ci = blocks
        a.row_ptr, a.col_idx = rp.data_ptr(), ci.data_ptr()
        a.block = 128
        a.flags = flags
        if q_norm is not None:
            a.flags |= _lib.H3C_FUSE_PROLOGUE
            a.q_norm_weight, a.k_norm_weight = q_norm.data_ptr(), k_norm.data_ptr()
            a.eps = eps
            if rope_table is None:
                a.flags |= _lib.H3C_NO_ROPE
            else:
                a.rope_table = rope_table.data_ptr()
                a.rope_half = rope_table.shape[1]
        return a

    def attn_fwd(self, *, stream=None, **kw):
        a = self.attn_args(**kw)
        self._check(self.L.h3c_attn_fwd(self.ctx, C.byref(a), _stream_ptr(stream)))

    def attn_fwd_sync(self, *, stream=None, **kw):
        """attn_fwd, synchronise, and raise H3CError(H3C_ERR_TIMEOUT) if a
        bounded device wait gave up."""
        a = self.attn_args(**kw)
        self._check(self.L.h3c_attn_fwd_sync(self.ctx, C.byref(a), _stream_ptr(stream)))

    # ------------------------------------------------- sequence-sharded path
    @staticmethod
    def comm_unique_id() -> bytes:
        cid = _lib.CommId()
        _lib.check(_lib.load().h3c_comm_unique_id(C.byref(cid)), what="h3c_comm_unique_id")
        return C.string_at(C.addressof(cid), 128)  # all 128 bytes (the id holds NULs)

    def comm_init(self, unique_id: bytes, nranks: int, rank: int):
        if len(unique_id) != 128:
            raise ValueError("an NCCL unique id is 128 bytes")
        cid = _lib.CommId()
        C.memmove(C.addressof(cid), unique_id, 128)
        self._check(self.L.h3c_comm_init(self.ctx, C.byref(cid), nranks, rank))

    def attn_fwd_seqshard(self, *, stream=None, timeout_ms=None, **kw):
        """This rank's [S_r, H, D] shards in and out; ``seq_len`` is global.
        With ``timeout_ms`` the call also waits (bounded) for the exchange:
        a rank that does not take part raises H3CError(H3C_ERR_TIMEOUT) after
        the communicator is aborted, instead of hanging."""
        seq_len = kw.pop("seq_len")
        a = self.attn_args(**kw)
        a.seq_len = seq_len
        self._check(self.L.h3c_attn_fwd_seqshard(self.ctx, C.byref(a), _stream_ptr(stream)))
        if timeout_ms is not None:
            self.comm_wait(stream, timeout_ms)

    def comm_wait(self, stream=None, timeout_ms: int = 60000):
        self._check(self.L.h3c_comm_wait(self.ctx, _stream_ptr(stream), int(timeout_ms)))

    def comm_destroy(self):
        self._check(self.L.h3c_comm_destroy(self.ctx))

    def device_status(self):
        self._check(self.L.h3c_device_status(self.ctx))

    def attn_fwd_args(self, a: _lib.AttnArgs, stream=None):
        self._check(self.L.h3c_attn_fwd(self.ctx, C.byref(a), _stream_ptr(stream)))

    # --------------------------------------------------------- conditioning
    def _launch(self, call, args, size_call, selector, stream):
        """Run ``call`` with workspace of the size ``size_call`` gives, taken
        from torch's allocator on the launching stream (so a captured call
        keeps its own, and the memory is not reused before the call is done)."""
        import torch

        need, why = C.c_size_t(0), C.create_string_buffer(256)
        st = size_call(C.byref(args), selector, C.byref(need), why, 256)
        if st != _lib.H3C_OK:
            raise _lib.H3CError(st, why.value.decode())
        if stream is None:
            stream = torch.cuda.current_stream(self.device)
        ws = None
        if need.value:
            with torch.cuda.stream(stream):
                ws = torch.empty(need.value, dtype=torch.uint8, device=f"cuda:{self.device}")
            args.workspace, args.workspace_bytes = ws.data_ptr(), need.value
        self._check(call(self.ctx, C.byref(args), stream.cuda_stream or None))

    def _cross_args(self, q, k, v, out, layout, scale, kv_lens, lse):
        import torch

        a, dev = _lib.CrossArgs(), self.device
        a.q, (B, S, H) = _bview("q", q, layout, dev)
        a.out, _ = _bview("out", out, layout, dev, (B, S, H))
        a.k, (kb, n, Hk) = _bview("k", k, layout, dev)
        if kb != B:
            raise ValueError(f"k must have the {B} members of q, got {kb}")
        a.v, _ = _bview("v", v, layout, dev, (B, n, Hk))
        a.batch, a.q_len, a.kv_len, a.heads, a.kv_heads, a.head_dim = B, S, n, H, Hk, 128
        a.scale = scale
        if kv_lens is not None:
            a.kv_lens = _vector("kv_lens", kv_lens, torch.int32, (B,), dev)
        if lse is not None:
            shape = (B, H, S) if q.dim() == 4 or lse.dim() == 3 else (H, S)
            a.lse = _vector("lse", lse, torch.float32, shape, dev)
        return a

    def cross_attn_fwd(self, *, q, k, v, out, scale, layout="SHD", kv_lens=None, lse=None, stream=None):
        """``out = softmax(scale q k^T) v`` against encoder states of another
        length.  q, out: [B, S, H, 128]; k, v: [B, N, Hk, 128] (or without
        B; "HSD": [B, H, S, 128]), H a multiple of Hk.  kv_lens: int32 [B]
        device tensor, the valid keys of each member; a member without keys
        gives zeros.  lse: optional fp32 [B, H, S] result, needed by
        ``cross_attn_bwd``."""
        a = self._cross_args(q, k, v, out, layout, scale, kv_lens, lse)
        self._launch(self.L.h3c_cross_attn_fwd, a, self.L.h3c_cross_workspace_size, _lib.H3C_OP_CROSS_FWD, stream)

    def cross_attn_bwd(self, *, q, k, v, out, lse, out_grad, dq, dk, dv, scale, layout="SHD", kv_lens=None,
                       stream=None):
        """Gradients of ``cross_attn_fwd``: dq as q, dk and dv as k (summed
        over the query heads of each key head, 0 past kv_lens), from the
        forward call's out and lse.  Deterministic."""
        a, dev = self._cross_args(q, k, v, out, layout, scale, kv_lens, lse), self.device
        mine, keys = (a.batch, a.q_len, a.heads), (a.batch, a.kv_len, a.kv_heads)
        a.out_grad, _ = _bview("out_grad", out_grad, layout, dev, mine)
        a.dq, _ = _bview("dq", dq, layout, dev, mine)
        a.dk, _ = _bview("dk", dk, layout, dev, keys)
        a.dv, _ = _bview("dv", dv, layout, dev, keys)
        self._launch(self.L.h3c_cross_attn_bwd, a, self.L.h3c_cross_workspace_size, _lib.H3C_OP_CROSS_BWD, stream)

    def prefix_attn_fwd(self, *, q, prefix_k, prefix_v, k, v, out, scale, layout="SHD", kv_lens=None, lse=None,
                        stream=None):
        """Attention of every member's queries over the keys all members
        share (prefix_k, prefix_v: [P, Hk, 128], "HSD": [Hk, P, 128]) and
        then its own, as ``cross_attn_fwd``."""
        a, dev = self._cross_args(q, k, v, out, layout, scale, kv_lens, lse), self.device
        if prefix_k.dim() != 3 or prefix_v.dim() != 3:
            raise ValueError("prefix_k and prefix_v have no batch axis")
        pk, (_, P, _) = _bview("prefix_k", prefix_k, layout, dev)
        _bview("prefix_k", prefix_k, layout, dev, (1, P, a.kv_heads))
        pv, _ = _bview("prefix_v", prefix_v, layout, dev, (1, P, a.kv_heads))
        a.prefix_k = _lib.View(pk.ptr, pk.token_stride, pk.head_stride)
        a.prefix_v = _lib.View(pv.ptr, pv.token_stride, pv.head_stride)
        a.prefix_len = P
        self._launch(self.L.h3c_prefix_attn_fwd, a, self.L.h3c_cross_workspace_size, _lib.H3C_OP_PREFIX_FWD, stream)

    def _rope_rows(self, name, table, batch, tokens):
        """(pointer, half, batch stride) of a bf16 [S, half, 4] or [B, S, half, 4] table."""
        import torch

        if table is None:
            return None, 0, 0
        shape = (tokens,) if table.dim() == 3 else (batch, tokens)
        if table.dtype is not torch.bfloat16 or table.device.type != "cuda" or table.device.index != self.device \
                or table.dim() not in (3, 4) or table.shape[-1] != 4 or tuple(table.shape[:-2]) != shape \
                or not table.is_contiguous():
            raise ValueError(f"{name} must be a contiguous bfloat16 {(*shape, 'half', 4)} tensor on cuda:{self.device}, "
                             f"got {table.dtype} {tuple(table.shape)} on {table.device}")
        return table.data_ptr(), table.shape[-2], tokens * table.shape[-2] * 4 if table.dim() == 4 else 0

    def _norm_args(self, q, k, q_norm, k_norm, eps, q_rope, k_rope, layout):
        import torch

        a, dev = _lib.QkNormArgs(), self.device
        a.q, (B, S, H) = _bview("q", q, layout, dev)
        a.k, (kb, n, Hk) = _bview("k", k, layout, dev)
        if kb != B:
            raise ValueError(f"k must have the {B} members of q, got {kb}")
        a.batch, a.q_len, a.k_len, a.heads, a.kv_heads, a.head_dim, a.eps = B, S, n, H, Hk, 128, eps
        a.q_norm_weight = _vector("q_norm", q_norm, torch.bfloat16, (128,), dev)
        a.k_norm_weight = _vector("k_norm", k_norm, torch.bfloat16, (128,), dev)
        a.q_rope, a.q_rope_half, a.q_rope_batch_stride = self._rope_rows("q_rope", q_rope, B, S)
        a.k_rope, a.k_rope_half, a.k_rope_batch_stride = self._rope_rows("k_rope", k_rope, B, n)
        return a

    def qk_norm_rope_fwd(self, *, q, k, q_out, k_out, q_norm, k_norm, eps=1e-6, q_rope=None, k_rope=None,
                         layout="SHD", stream=None):
        """Per-head RMSNorm of queries and keys and their rotation in one
        pass, fp32 with one rounding.  q: [B, S, H, 128], k: [B, N, Hk, 128];
        q_out / k_out may be q / k.  Tables: bf16 [S, half, 4] (as
        ``rope_table`` makes them) or [B, S, half, 4]; None: norm only."""
        a, dev = self._norm_args(q, k, q_norm, k_norm, eps, q_rope, k_rope, layout), self.device
        a.q_out, _ = _bview("q_out", q_out, layout, dev, (a.batch, a.q_len, a.heads))
        a.k_out, _ = _bview("k_out", k_out, layout, dev, (a.batch, a.k_len, a.kv_heads))
        if stream is None:
            import torch

            stream = torch.cuda.current_stream(dev)
        self._check(self.L.h3c_qk_norm_rope_fwd(self.ctx, C.byref(a), stream.cuda_stream or None))

    def qk_norm_rope_bwd(self, *, q, k, q_grad, k_grad, q_norm, k_norm, dq, dk, dq_norm, dk_norm, eps=1e-6,
                         q_rope=None, k_rope=None, layout="SHD", stream=None):
        """Gradients of ``qk_norm_rope_fwd`` from those of its outputs
        (q_grad, k_grad): dq, dk (may be q_grad, k_grad) and the fp32 [128]
        gradients of the two weights.  Deterministic."""
        import torch

        a, dev = self._norm_args(q, k, q_norm, k_norm, eps, q_rope, k_rope, layout), self.device
        mine, keys = (a.batch, a.q_len, a.heads), (a.batch, a.k_len, a.kv_heads)
        a.q_grad, _ = _bview("q_grad", q_grad, layout, dev, mine)
        a.k_grad, _ = _bview("k_grad", k_grad, layout, dev, keys)
        a.dq, _ = _bview("dq", dq, layout, dev, mine)
        a.dk, _ = _bview("dk", dk, layout, dev, keys)
        a.q_norm_grad = _vector("dq_norm", dq_norm, torch.float32, (128,), dev)
        a.k_norm_grad = _vector("dk_norm", dk_norm, torch.float32, (128,), dev)
        self._launch(self.L.h3c_qk_norm_rope_bwd, a, self.L.h3c_qk_norm_workspace_size, 1, stream)

    # ------------------------------------------------------------- prologue
    def prologue(self, x, out, weight, eps, rope_table=None, layout="SHD", stream=None):
        seq_axis = 0 if layout == "SHD" else 1
        S, H = x.shape[seq_axis], x.shape[1 - seq_axis]
        half = rope_table.shape[1] if rope_table is not None else 0
        self._check(self.L.h3c_prologue(self.ctx, view_of(x, layout), view_of(out, layout), S, H, 0, H,
                                        weight.data_ptr(), eps,
                                        rope_table.data_ptr() if rope_table is not None else None, half,
                                        _stream_ptr(stream)))

    def rope_table(self, pos, dims=(32, 48, 48), theta=1e4, stream=None):
        import torch

        S = pos.shape[0]
        half = sum(dims) // 2
        out = torch.empty((S, half, 4), dtype=torch.bfloat16, device=pos.device)
        d = (C.c_int32 * 3)(*dims)
        self._check(self.L.h3c_rope_table(self.ctx, pos.data_ptr(), S, d, theta, out.data_ptr(),
                                          _stream_ptr(stream)))
        return out

    def rope_table_shared(self, pos, inv_freq, stream=None):
        """The production table: float positions [S, 3] and the shared
        inv_freq [n] (both fp32 on this device); returns bf16 [S, 3n, 4]."""
        import torch

        pos = pos.to(torch.float32).contiguous()
        inv = inv_freq.to(device=pos.device, dtype=torch.float32).contiguous()
        S, n = pos.shape[0], inv.shape[0]
        out = torch.empty((S, 3 * n, 4), dtype=torch.bfloat16, device=pos.device)
        self._check(self.L.h3c_rope_table_shared(self.ctx, pos.data_ptr(), S, inv.data_ptr(), n, out.data_ptr(),
                                                 _stream_ptr(stream)))
        return out

    def fill_normal(self, out, seed, stream_id, mean=0.0, std=1.0, stream=None):
        self._check(self.L.h3c_fill_normal_bf16(self.ctx, out.data_ptr(), out.numel(), seed, stream_id, mean, std,
                                                _stream_ptr(stream)))
        return out

    def validate_blocks(self, blocks, stream=None):
        """Check a device block list (row_ptr [n_blocks+1], col_idx [nnz]
        int32 tensors on this device): row_ptr starts at 0, never decreases
        and ends at nnz; columns in [0, n_blocks), strictly ascending per
        row.  Raises H3CError(H3C_ERR_INVALID_ARGUMENT) with the reason.
        Synchronises the stream."""
        rp, ci = blocks
        self._check(self.L.h3c_blockmask_validate(self.ctx, rp.data_ptr(), ci.data_ptr(), rp.numel() - 1, ci.numel(),
                                                  _stream_ptr(stream)))

    def blockmask_device(self, spec, capacity: int, stream=None):
        import torch

        nb = spec.n_blocks
        rp = torch.empty(nb + 1, dtype=torch.int32, device=f"cuda:{self.device}")
        ci = torch.empty(max(capacity, 1), dtype=torch.int32, device=f"cuda:{self.device}")
        nnz = C.c_int64(0)
        cs = spec.to_c()
        self._check(self.L.h3c_blockmask_build_device(self.ctx, C.byref(cs), rp.data_ptr(), ci.data_ptr(), ci.numel(),
                                                      C.byref(nnz), _stream_ptr(stream)))
        return rp, ci[: nnz.value]
