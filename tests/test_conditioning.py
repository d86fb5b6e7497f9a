"""Refusals of the conditioning calls (cross attention, shared prefix, q/k
norm), on CPU: the checks run on the host before anything is launched."""
import ctypes as C

import pytest

PTR = 1 << 20  # never dereferenced


@pytest.fixture(scope="module")
def lib():
    from h3attention import _lib

    _lib.load()
    return _lib


def _view(lib, tokens, heads, ptr=PTR):
    return lib.BView(ptr, tokens * heads * 128, heads * 128, 128)


def _cross(lib, batch=2, q_len=5, kv_len=7, heads=4, kv_heads=2, prefix_len=3):
    a = lib.CrossArgs()
    a.batch, a.q_len, a.kv_len, a.heads, a.kv_heads, a.head_dim = batch, q_len, kv_len, heads, kv_heads, 128
    a.scale, a.prefix_len, a.lse = 0.1, prefix_len, PTR
    for n in ("q", "out", "out_grad", "dq"):
        setattr(a, n, _view(lib, q_len, heads))
    for n in ("k", "v", "dk", "dv"):
        setattr(a, n, _view(lib, kv_len, kv_heads))
    a.prefix_k = a.prefix_v = lib.View(PTR, kv_heads * 128, 128)
    return a


def _norm(lib, batch=2, q_len=5, k_len=7, heads=4, kv_heads=2):
    a = lib.QkNormArgs()
    a.batch, a.q_len, a.k_len, a.heads, a.kv_heads, a.head_dim, a.eps = batch, q_len, k_len, heads, kv_heads, 128, 1e-6
    for n in ("q", "q_out", "q_grad", "dq"):
        setattr(a, n, _view(lib, q_len, heads))
    for n in ("k", "k_out", "k_grad", "dk"):
        setattr(a, n, _view(lib, k_len, kv_heads))
    a.q_norm_weight = a.k_norm_weight = a.q_rope = a.k_rope = a.q_norm_grad = a.k_norm_grad = PTR
    a.q_rope_half = a.k_rope_half = 64
    return a


def _ask(lib, a, selector):
    n, why = C.c_size_t(7), C.create_string_buffer(256)
    call = lib.load().h3c_cross_workspace_size if isinstance(a, lib.CrossArgs) else lib.load().h3c_qk_norm_workspace_size
    return call(C.byref(a), selector, C.byref(n), why, 256), n.value, why.value.decode()


def _set(path, value):
    def change(a):
        *outer, last = path.split(".")
        o = a
        for n in outer:
            o = getattr(o, n)
        setattr(o, last, value)
    return change


INVALID, UNSUPPORTED = 1, 2
CROSS = [
    ("head_dim", 64, UNSUPPORTED, "head_dim", (0, 1, 2)),
    ("kv_heads", 3, INVALID, "multiple", (0, 1, 2)),
    ("heads", 0, INVALID, "heads", (0, 1, 2)),
    ("batch", -1, INVALID, "batch", (0, 1, 2)),
    ("q_len", -1, INVALID, "lengths", (0, 1, 2)),
    ("kv_len", -5, INVALID, "lengths", (0, 1, 2)),
    ("scale", 0.0, INVALID, "scale", (0, 1, 2)),
    ("scale", float("nan"), INVALID, "scale", (0, 1, 2)),
    ("scale", float("inf"), INVALID, "scale", (0, 1, 2)),
    ("q.ptr", None, INVALID, "q is null", (0, 1, 2)),
    ("v.ptr", PTR + 8, UNSUPPORTED, "v needs 16-byte", (0, 1, 2)),
    ("k.token_stride", 0, UNSUPPORTED, "k is broadcast", (0, 1, 2)),
    ("k.batch_stride", 132, UNSUPPORTED, "k needs 16-byte", (0, 1, 2)),
    ("q.head_stride", -128, INVALID, "negative", (0, 1, 2)),
    ("q.batch_stride", 1 << 39, UNSUPPORTED, "2^40", (0, 1, 2)),
    ("out.head_stride", 0, INVALID, "out overlaps itself", (0, 2)),
    ("out.token_stride", 128, INVALID, "out overlaps itself", (0, 2)),
    ("kv_lens", PTR + 2, UNSUPPORTED, "kv_lens", (0, 1, 2)),
    ("q_len", 1 << 30, UNSUPPORTED, "2^31", (0, 1, 2)),
    ("reserved", 1, INVALID, "reserved", (0, 1, 2)),
    ("lse", None, INVALID, "lse", (1,)),
    ("dk.batch_stride", 0, INVALID, "dk overlaps itself", (1,)),
    ("dq.ptr", None, INVALID, "dq is null", (1,)),
    ("prefix_len", -1, INVALID, "prefix_len", (2,)),
    ("prefix_k.ptr", None, INVALID, "prefix_k is null", (2,)),
]


@pytest.mark.parametrize("path,value,status,why,ops", CROSS, ids=[f"{c[0]}={c[1]}" for c in CROSS])
def test_cross_refusals(lib, path, value, status, why, ops):
    for op in (0, 1, 2):
        a = _cross(lib)
        assert _ask(lib, a, op)[0] == lib.H3C_OK
        _set(path, value)(a)
        st, n, said = _ask(lib, a, op)
        if op in ops:
            assert (st, n) == (status, 0) and why in said, said
        else:
            assert st == lib.H3C_OK, said


def test_cross_allows(lib):
    for change in (_set("k.batch_stride", 0), _set("v.head_stride", 0), _set("lse", None), _set("kv_lens", PTR)):
        a = _cross(lib)
        change(a)
        assert _ask(lib, a, 0)[0] == lib.H3C_OK
    a = _cross(lib, batch=1, q_len=1)  # strides of axes with one element are not read
    a.q.batch_stride = a.q.token_stride = a.out.batch_stride = a.out.token_stride = -3
    assert _ask(lib, a, 0)[0] == lib.H3C_OK
    a = _cross(lib, kv_len=0)
    a.k.ptr = a.v.ptr = a.dk.ptr = a.dv.ptr = None
    assert [_ask(lib, a, op)[0] for op in (0, 1, 2)] == [0, 0, 0]
    a = _cross(lib, batch=0)
    for n in ("q", "out", "k", "v"):
        getattr(a, n).ptr = None
    assert _ask(lib, a, 2) == (lib.H3C_OK, _ask(lib, a, 2)[1], "")
    assert _ask(lib, _cross(lib), 3)[0] == lib.H3C_ERR_INVALID_ARGUMENT
    assert _ask(lib, _cross(lib), -1)[0] == lib.H3C_ERR_INVALID_ARGUMENT


NORM = [
    ("head_dim", 96, UNSUPPORTED, "head_dim", (0, 1)),
    ("heads", -1, INVALID, "heads", (0, 1)),
    ("k_len", -1, INVALID, "lengths", (0, 1)),
    ("eps", -1e-6, INVALID, "eps", (0, 1)),
    ("eps", float("nan"), INVALID, "eps", (0, 1)),
    ("q_norm_weight", None, INVALID, "weights", (0, 1)),
    ("k_norm_weight", PTR + 8, UNSUPPORTED, "norm weights", (0, 1)),
    ("k_rope", PTR + 4, UNSUPPORTED, "rope tables", (0, 1)),
    ("q_rope_half", 65, UNSUPPORTED, "half", (0, 1)),
    ("k_rope_half", 0, UNSUPPORTED, "half", (0, 1)),
    ("q_rope_batch_stride", 2, INVALID, "batch stride", (0, 1)),
    ("q.ptr", None, INVALID, "q is null", (0, 1)),
    ("k.token_stride", 260, UNSUPPORTED, "k needs 16-byte", (0, 1)),
    ("k_out.head_stride", 0, INVALID, "k_out overlaps itself", (0,)),
    ("dq.token_stride", 0, INVALID, "dq overlaps itself", (1,)),
    ("k_grad.ptr", None, INVALID, "k_grad is null", (1,)),
    ("q_norm_grad", None, INVALID, "q_norm_grad", (1,)),
    ("reserved", 2, INVALID, "reserved", (0, 1)),
]


@pytest.mark.parametrize("path,value,status,why,ops", NORM, ids=[f"{c[0]}={c[1]}" for c in NORM])
def test_norm_refusals(lib, path, value, status, why, ops):
    for op in (0, 1):
        a = _norm(lib)
        assert _ask(lib, a, op)[0] == lib.H3C_OK
        _set(path, value)(a)
        st, n, said = _ask(lib, a, op)
        if op in ops:
            assert (st, n) == (status, 0) and why in said, said
        else:
            assert st == lib.H3C_OK, said


def test_sizes_whose_products_pass_64_bits(lib):
    """2^31 - 1 on three axes: 2^93 rows must not wrap to a number that passes."""
    big = 2 ** 31 - 1
    for a in (_cross(lib), _norm(lib)):
        a.batch = a.heads = a.kv_heads = a.q_len = big
        for op in (0, 1):
            st, n, said = _ask(lib, a, op)
            assert (st, n) == (lib.H3C_ERR_UNSUPPORTED, 0) and "2^31 rows" in said, said
    a = _cross(lib, batch=1, kv_len=2 ** 20)
    for v in (a.k, a.v, a.dk, a.dv):
        v.token_stride = 2 ** 38
    st, _, said = _ask(lib, a, 1)
    assert st == lib.H3C_ERR_UNSUPPORTED and "dk spans 2^47 bytes" in said, said


def test_null_arguments(lib):
    L = lib.load()
    n = C.c_size_t()
    assert L.h3c_cross_workspace_size(None, 0, C.byref(n), None, 0) == lib.H3C_ERR_INVALID_ARGUMENT
    assert L.h3c_cross_workspace_size(C.byref(_cross(lib)), 0, None, None, 0) == lib.H3C_ERR_INVALID_ARGUMENT
    assert L.h3c_qk_norm_workspace_size(None, 1, C.byref(n), None, 0) == lib.H3C_ERR_INVALID_ARGUMENT
    for call in (L.h3c_cross_attn_fwd, L.h3c_cross_attn_bwd, L.h3c_prefix_attn_fwd):
        assert call(None, C.byref(_cross(lib)), None) == lib.H3C_ERR_INVALID_ARGUMENT
    for call in (L.h3c_qk_norm_rope_fwd, L.h3c_qk_norm_rope_bwd):
        assert call(None, C.byref(_norm(lib)), None) == lib.H3C_ERR_INVALID_ARGUMENT


def test_struct_sizes_match_the_header(lib, tmp_path):
    """sizeof and field offsets as the C compiler lays the header out."""
    import os
    import subprocess

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    fields = [("h3c_cross_args", lib.CrossArgs), ("h3c_qk_norm_args", lib.QkNormArgs), ("h3c_bview", lib.BView)]
    src = tmp_path / "s.c"
    src.write_text('#include "h3cuda.h"\n#include <stdio.h>\nint main(void) {\n' + "".join(
        f'printf("%zu\\n", sizeof({c}));\n' + "".join(f'printf("%zu\\n", offsetof({c}, {f[0]}));\n' for f in t._fields_)
        for c, t in fields) + "return 0;}\n")
    exe = tmp_path / "s"
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    want = [x for _, t in fields for x in (C.sizeof(t), *(getattr(t, f[0]).offset for f in t._fields_))]
    assert got == want


def test_packed_arguments_match_the_structures(lib):
    """The Python calls pack their arguments; every field lands where ctypes has it."""
    from h3attention.runtime import _CROSS, _NORM

    for packer, cls in ((_CROSS, lib.CrossArgs), (_NORM, lib.QkNormArgs)):
        assert packer.size == C.sizeof(cls)
        flat = []

        def collect(o):
            for name, t in o._fields_:
                v = getattr(o, name)
                if isinstance(v, C.Structure):
                    collect(v)
                else:
                    flat.append(t)

        collect(cls())
        values = [float(i) if t is C.c_float else i for i, t in enumerate(flat, 1)]
        a, got = cls.from_buffer_copy(packer.pack(*values)), []

        def read(o):
            for name, _ in o._fields_:
                v = getattr(o, name)
                read(v) if isinstance(v, C.Structure) else got.append(v)

        read(a)
        assert got == values


def test_python_refuses_host_tensors_and_types(lib):
    """The tensor checks of the Python calls run before the library is entered."""
    import torch

    from h3attention.runtime import _axes, _check_vector, _cross_workspace, _kind, _norm_workspace

    with pytest.raises(ValueError, match="must be bfloat16 on cuda:0"):
        _axes("q", _kind(torch.zeros(2, 3, 128, dtype=torch.bfloat16)), False, 0)
    with pytest.raises(ValueError, match="must be a contiguous"):
        _check_vector("kv_lens", _kind(torch.zeros(2, dtype=torch.int64)), torch.int32, (2,), 0)
    a = _cross(lib)
    for op in (0, 1, 2):
        assert _cross_workspace(op, 2, 5, 7, 3, 4, 2) == _ask(lib, a, op)[1]
    assert _norm_workspace() == _ask(lib, _norm(lib), 1)[1] > 0


def test_cross_sdpa_refuses_host_tensors():
    import torch

    from h3attention import cross_sdpa

    x = torch.zeros(3, 2, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="must be a CUDA tensor"):
        cross_sdpa(x, x, x, 128)
