"""Per-device handle on the C ABI: one ``h3c_ctx`` per CUDA device.

Torch tensors are accepted for convenience; only their device pointers,
shapes and strides cross the boundary.
"""
from __future__ import annotations

import ctypes as C
import functools
import struct
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


# h3c_cross_args and h3c_qk_norm_args, packed in one call: a small operator's
# time is mostly that of its Python call, and filling the ctypes structures
# field by field took 12 of its 20 us.
_CROSS = struct.Struct("@" + "Pqqq" * 4 + "6if" + "PP" + "Pqq" * 2 + "ii" + "Pqqq" * 4 + "PN")
_NORM = struct.Struct("@" + "Pqqq" * 4 + "6i" + "4P" + "qq" + "iifi" + "Pqqq" * 4 + "PPPN")
_NO_ROWS = (0, 0, 0, 0)


def _kind(t):
    """What a check of a tensor goes by."""
    return t.shape, t.stride(), t.dtype, t.get_device()


def _axes(name, kind, hsd: bool, device: int, want=None):
    """``((batch, token and head stride), (batch, tokens, heads))`` of a bf16
    tensor on ``device``: [B, S, H, 128] or [S, H, 128], with ``hsd``
    [B, H, S, 128] or [H, S, 128].  ``want``: the (batch, tokens, heads) it
    must have."""
    import torch

    size, stride, dtype, where = kind
    if dtype is not torch.bfloat16 or where != device:
        raise ValueError(f"{name} must be bfloat16 on cuda:{device}, got {dtype} on "
                         f"{'the host' if where < 0 else f'cuda:{where}'}")
    if len(size) == 4:
        (b, s, h, d), (sb, ss, sh, sd) = size, stride
    elif len(size) == 3:
        (s, h, d), (ss, sh, sd), b, sb = size, stride, 1, 0
    else:
        raise ValueError(f"{name} must have 3 or 4 axes, got {tuple(size)}")
    if hsd:
        s, h, ss, sh = h, s, sh, ss
    if sd != 1 and d > 1:
        raise ValueError(f"{name}: head_dim must be contiguous")
    if d != 128:
        raise _lib.H3CError(_lib.H3C_ERR_UNSUPPORTED, f"{name}: head_dim must be 128, got {d}")
    if want is not None and (b, s, h) != want:
        raise ValueError(f"{name} must have {want} (batch, tokens, heads), got {(b, s, h)}")
    return (sb, ss, sh), (b, s, h)


# The checks of a call's operands and what follows from their shapes, strides,
# types and device alone: a program makes the same call again and again, and
# going through them took 3 of its 8 us in Python.
@functools.lru_cache(maxsize=4096)
def _cross_form(op, hsd, device, q, out, k, v, lens, lse, prefix, grads):
    """Strides and sizes of a call, in the order of its arguments."""
    import torch

    aq, mine = _axes("q", q, hsd, device)
    ao, _ = _axes("out", out, hsd, device, mine)
    ak, keys = _axes("k", k, hsd, device)
    av, _ = _axes("v", v, hsd, device, keys)
    (B, S, H), (_, N, Hk) = mine, keys
    if keys[0] != B:
        raise ValueError(f"k must have the {B} members of q, got {keys[0]}")
    if lens is not None:
        _check_vector("kv_lens", lens, torch.int32, (B,), device)
    if lse is not None:
        _check_vector("lse", lse, torch.float32, (B, H, S) if len(lse[0]) == 3 or B > 1 else (H, S), device)
    P, ap = 0, ((0, 0), (0, 0))
    if prefix is not None:
        if len(prefix[0][0]) != 3 or len(prefix[1][0]) != 3:
            raise ValueError("prefix_k and prefix_v have no batch axis")
        (_, pks, pkh), (_, P, ph) = _axes("prefix_k", prefix[0], hsd, device)
        (_, pvs, pvh), _ = _axes("prefix_v", prefix[1], hsd, device, (1, P, ph))
        if ph != Hk:
            raise ValueError(f"prefix_k must have the {Hk} heads of k, got {ph}")
        ap = ((pks, pkh), (pvs, pvh))
    ag = ((0, 0, 0),) * 4
    if grads is not None:
        ag = tuple(_axes(n, g, hsd, device, w)[0]
                   for n, g, w in zip(("out_grad", "dq", "dk", "dv"), grads, (mine, mine, keys, keys)))
    return aq, ao, ak, av, ap, ag, (B, S, N, H, Hk, 128), P, _cross_workspace(op, B, S, N, P, H, Hk)


@functools.lru_cache(maxsize=4096)
def _norm_form(hsd, device, q, k, yq, yk, q_norm, k_norm, q_rope, k_rope, grads):
    import torch

    aq, mine = _axes("q", q, hsd, device)
    ak, keys = _axes("k", k, hsd, device)
    if keys[0] != mine[0]:
        raise ValueError(f"k must have the {mine[0]} members of q, got {keys[0]}")
    names = ("q_out", "k_out") if grads is None else ("dq", "dk")
    ayq, _ = _axes(names[0], yq, hsd, device, mine)
    ayk, _ = _axes(names[1], yk, hsd, device, keys)
    _check_vector("q_norm", q_norm, torch.bfloat16, (128,), device)
    _check_vector("k_norm", k_norm, torch.bfloat16, (128,), device)
    hq, bq = _rope_form("q_rope", q_rope, mine[0], mine[1], device)
    hk, bk = _rope_form("k_rope", k_rope, mine[0], keys[1], device)
    ag = None
    if grads is not None:
        ag = _axes("q_grad", grads[0], hsd, device, mine)[0], _axes("k_grad", grads[1], hsd, device, keys)[0]
        _check_vector("dq_norm", grads[2], torch.float32, (128,), device)
        _check_vector("dk_norm", grads[3], torch.float32, (128,), device)
    return aq, ak, ayq, ayk, ag, (mine[0], mine[1], keys[1], mine[2], keys[2], 128), (bq, bk, hq, hk)


def _contiguous(size, stride) -> bool:
    if 0 in size:
        return True
    n = 1
    for axis, step in zip(reversed(size), reversed(stride)):
        if axis != 1 and step != n:
            return False
        n *= axis
    return True


def _check_vector(name, kind, dtype, shape, device: int) -> None:
    """Refuses what is not a contiguous tensor of the given type and shape."""
    size, stride, given, where = kind
    if given is not dtype or where != device or size != shape or not _contiguous(size, stride):
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {shape} on cuda:{device}, got "
                         f"{given} {tuple(size)} on {'the host' if where < 0 else f'cuda:{where}'}")


def _rope_form(name, kind, batch: int, tokens: int, device: int):
    """(half, batch stride) of a bf16 [S, half, 4] or [B, S, half, 4] table."""
    import torch

    if kind is None:
        return 0, 0
    shape, stride, dtype, where = kind
    each = len(shape) == 4
    if dtype is not torch.bfloat16 or where != device or not 3 <= len(shape) <= 4 or shape[-1] != 4 \
            or shape[:-2] != ((batch, tokens) if each else (tokens,)) or not _contiguous(shape, stride):
        raise ValueError(f"{name} must be a contiguous bfloat16 [{tokens}, half, 4] or [{batch}, {tokens}, half, 4] "
                         f"tensor on cuda:{device}, got {dtype} {tuple(shape)} on "
                         f"{'the host' if where < 0 else f'cuda:{where}'}")
    return shape[-2], tokens * shape[-2] * 4 if each else 0


def _hsd(layout: str) -> bool:
    if layout != "SHD" and layout != "HSD":
        raise ValueError(layout)
    return layout == "HSD"


@functools.lru_cache(maxsize=4096)
def _cross_workspace(op, batch, q_len, kv_len, prefix_len, heads, kv_heads) -> int:
    """Bytes of workspace of a call of these sizes.  It depends on nothing
    else, so the operands are stood in for by aligned pointers; a call whose
    sizes are refused is refused by itself."""
    a, n = _lib.CrossArgs(), C.c_size_t(0)
    a.batch, a.q_len, a.kv_len, a.heads, a.kv_heads, a.head_dim = batch, q_len, kv_len, heads, kv_heads, 128
    a.scale, a.lse, a.prefix_len = 1.0, 256, prefix_len
    for names, s, h in ((("q", "out", "out_grad", "dq"), q_len, heads), (("k", "v", "dk", "dv"), kv_len, kv_heads)):
        for name in names:
            setattr(a, name, _lib.BView(256, s * h * 128, h * 128, 128))
    a.prefix_k = a.prefix_v = _lib.View(256, kv_heads * 128, 128)
    _lib.load().h3c_cross_workspace_size(C.byref(a), op, C.byref(n), None, 0)
    return n.value


@functools.lru_cache(maxsize=None)
def _norm_workspace() -> int:
    a, n = _lib.QkNormArgs(), C.c_size_t(0)
    a.heads = a.kv_heads = 1
    a.head_dim, a.q_norm_weight, a.k_norm_weight, a.q_norm_grad, a.k_norm_grad = 128, 256, 256, 256, 256
    _lib.check(_lib.load().h3c_qk_norm_workspace_size(C.byref(a), 1, C.byref(n), None, 0), what="workspace size")
    return n.value


class Runtime:
    _lock = threading.Lock()
    _by_device: Dict[int, "Runtime"] = {}

    def __init__(self, device: int):
        self.L = _lib.load()
        self._packed = _lib.load_packed()
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
    def _workspace(self, size: int, stream):
        """Scratch from torch's allocator on the launching stream (None: the
        current one), so a captured call keeps its own and the memory is not
        reused before the call is done."""
        import torch

        if stream is None:
            return torch.empty(size, dtype=torch.uint8, device=self._torch_device)
        with torch.cuda.stream(stream):
            return torch.empty(size, dtype=torch.uint8, device=self._torch_device)

    @functools.cached_property
    def _torch_device(self):
        import torch

        return torch.device("cuda", self.device)

    def _launch(self, call, args, stream):
        """A conditioning call on ``stream`` (None: the device's current one,
        asked for by its handle alone: a Stream object takes 1.3 us to make)."""
        import torch

        status = call(self.ctx, args, torch._C._cuda_getCurrentRawStream(self.device) if stream is None
                      else stream.cuda_stream)
        if status:
            self._check(status)

    def _cross(self, op, call, q, k, v, out, layout, scale, kv_lens, lse, stream, prefix=None, grads=None):
        aq, ao, ak, av, (apk, apv), ag, sizes, P, size = _cross_form(
            op, _hsd(layout), self.device, _kind(q), _kind(out), _kind(k), _kind(v),
            None if kv_lens is None else _kind(kv_lens), None if lse is None else _kind(lse),
            None if prefix is None else (_kind(prefix[0]), _kind(prefix[1])),
            None if grads is None else tuple(_kind(g) for g in grads))
        lens = 0 if kv_lens is None else kv_lens.data_ptr()
        plse = 0 if lse is None else lse.data_ptr()
        ws = self._workspace(size, stream) if size else None
        pk, pv = (0, 0) if prefix is None else (prefix[0].data_ptr(), prefix[1].data_ptr())
        g0, g1, g2, g3 = (0, 0, 0, 0) if grads is None else (g.data_ptr() for g in grads)
        args = _CROSS.pack(q.data_ptr(), *aq, out.data_ptr(), *ao, k.data_ptr(), *ak, v.data_ptr(), *av, *sizes, scale,
                           lens, plse, pk, *apk, pv, *apv, P, 0, g0, *ag[0], g1, *ag[1], g2, *ag[2], g3, *ag[3],
                           ws.data_ptr() if size else 0, size)
        self._launch(call, args, stream)

    def cross_attn_fwd(self, *, q, k, v, out, scale, layout="SHD", kv_lens=None, lse=None, stream=None):
        """``out = softmax(scale q k^T) v`` against encoder states of another
        length.  q, out: [B, S, H, 128]; k, v: [B, N, Hk, 128] (or without
        B; "HSD": [B, H, S, 128]), H a multiple of Hk.  kv_lens: int32 [B]
        device tensor, the valid keys of each member; a member without keys
        gives zeros.  lse: optional fp32 [B, H, S] result, needed by
        ``cross_attn_bwd``."""
        self._cross(_lib.H3C_OP_CROSS_FWD, self._packed.h3c_cross_attn_fwd, q, k, v, out, layout, scale, kv_lens, lse,
                    stream)

    def cross_attn_bwd(self, *, q, k, v, out, lse, out_grad, dq, dk, dv, scale, layout="SHD", kv_lens=None,
                       stream=None):
        """Gradients of ``cross_attn_fwd``: dq as q, dk and dv as k (summed
        over the query heads of each key head, 0 past kv_lens), from the
        forward call's out and lse.  Deterministic."""
        self._cross(_lib.H3C_OP_CROSS_BWD, self._packed.h3c_cross_attn_bwd, q, k, v, out, layout, scale, kv_lens, lse,
                    stream, grads=(out_grad, dq, dk, dv))

    def prefix_attn_fwd(self, *, q, prefix_k, prefix_v, k, v, out, scale, layout="SHD", kv_lens=None, lse=None,
                        stream=None):
        """Attention of every member's queries over the keys all members
        share (prefix_k, prefix_v: [P, Hk, 128], "HSD": [Hk, P, 128]) and
        then its own, as ``cross_attn_fwd``."""
        self._cross(_lib.H3C_OP_PREFIX_FWD, self._packed.h3c_prefix_attn_fwd, q, k, v, out, layout, scale, kv_lens,
                    lse, stream, prefix=(prefix_k, prefix_v))

    def _norm(self, call, q, k, outs, q_norm, k_norm, eps, q_rope, k_rope, layout, stream, grads=None):
        yq, yk = outs if grads is None else grads[2:4]
        aq, ak, ayq, ayk, ag, sizes, ropes = _norm_form(
            _hsd(layout), self.device, _kind(q), _kind(k), _kind(yq), _kind(yk), _kind(q_norm), _kind(k_norm),
            None if q_rope is None else _kind(q_rope), None if k_rope is None else _kind(k_rope),
            None if grads is None else tuple(_kind(grads[i]) for i in (0, 1, 4, 5)))
        yq, yk = (yq.data_ptr(), *ayq), (yk.data_ptr(), *ayk)
        size, ws, fwd, back, dw = 0, None, (yq, yk), (_NO_ROWS,) * 4, (0, 0)
        if grads is not None:
            size = _norm_workspace()
            ws = self._workspace(size, stream)
            dw = grads[4].data_ptr(), grads[5].data_ptr()
            fwd = (_NO_ROWS, _NO_ROWS)
            back = (grads[0].data_ptr(), *ag[0]), yq, (grads[1].data_ptr(), *ag[1]), yk
        args = _NORM.pack(q.data_ptr(), *aq, *fwd[0], k.data_ptr(), *ak, *fwd[1], *sizes, q_norm.data_ptr(),
                          k_norm.data_ptr(), 0 if q_rope is None else q_rope.data_ptr(),
                          0 if k_rope is None else k_rope.data_ptr(), *ropes, eps, 0, *back[0], *back[1], *back[2],
                          *back[3], *dw, ws.data_ptr() if size else 0, size)
        self._launch(call, args, stream)

    def qk_norm_rope_fwd(self, *, q, k, q_out, k_out, q_norm, k_norm, eps=1e-6, q_rope=None, k_rope=None,
                         layout="SHD", stream=None):
        """Per-head RMSNorm of queries and keys and their rotation in one
        pass, fp32 with one rounding.  q: [B, S, H, 128], k: [B, N, Hk, 128];
        q_out / k_out may be q / k.  Tables: bf16 [S, half, 4] (as
        ``rope_table`` makes them) or [B, S, half, 4]; None: norm only."""
        self._norm(self._packed.h3c_qk_norm_rope_fwd, q, k, (q_out, k_out), q_norm, k_norm, eps, q_rope, k_rope,
                   layout, stream)

    def qk_norm_rope_bwd(self, *, q, k, q_grad, k_grad, q_norm, k_norm, dq, dk, dq_norm, dk_norm, eps=1e-6,
                         q_rope=None, k_rope=None, layout="SHD", stream=None):
        """Gradients of ``qk_norm_rope_fwd`` from those of its outputs
        (q_grad, k_grad): dq, dk (may be q_grad, k_grad) and the fp32 [128]
        gradients of the two weights.  Deterministic."""
        self._norm(self._packed.h3c_qk_norm_rope_bwd, q, k, None, q_norm, k_norm, eps, q_rope, k_rope, layout, stream,
                   grads=(q_grad, k_grad, dq, dk, dq_norm, dk_norm))

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
