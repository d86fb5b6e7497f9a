"""Failure detection of the conditioning calls without a GPU fault: the host
has the producers skip one load of every block (a test hook read from the
environment), so that the bounded waits run out after a short limit.  The
context must report H3C_ERR_TIMEOUT and then give right results again."""
import contextlib

import pytest

import test_gpu_conditioning as base

pytestmark = pytest.mark.gpu


@contextlib.contextmanager
def _dropped(monkeypatch, item, limit_ns=50_000_000):
    with monkeypatch.context() as m:
        m.setenv("H3C_TEST_WAIT_LIMIT_NS", str(limit_ns))
        m.setenv("H3C_TEST_DROP_ITEM", str(item))
        yield


def _times_out():
    import torch

    from h3attention import H3CError, _lib

    torch.cuda.synchronize()
    with pytest.raises(H3CError, match="bounded device wait") as e:
        base._rt().device_status()
    assert e.value.status == _lib.H3C_ERR_TIMEOUT
    base._rt().device_status()  # cleared


# (batch, q_len, kv_len, heads, kv_heads, dropped load): a block's first load, one
# of a full ring, one that a later unit needs; every form of the kernels
CASES = [
    (2, 260, 300, 3, 3, 0), (1, 2000, 4096, 8, 8, 5),  # dense, short and long
    (40, 260, 300, 4, 4, 4),                           # dense, a second unit's
    (2, 4, 3000, 8, 4, 0), (16, 4, 3000, 8, 4, 4),     # single
    (3, 100, 1500, 8, 2, 0), (12, 100, 1500, 8, 2, 3), # dual
    (2, 300, 100, 4, 2, 0),                            # one block of keys
]


@pytest.mark.parametrize("B,S,N,H,Hk,item", CASES, ids=lambda x: str(x))
def test_dropped_load_of_cross_attention(gpu, monkeypatch, B, S, N, H, Hk, item):
    import torch

    q, k, v, do = base._inputs(B, S, N, H, Hk, 80)
    want = base._run_cross(q, k, v, None, do)
    with _dropped(monkeypatch, item):
        base._run_cross(q, k, v, None)
    _times_out()
    rt, lse = base._rt(), want["lse"]
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    with _dropped(monkeypatch, 0):
        rt.cross_attn_bwd(q=q, k=k, v=v, out=want["out"], lse=lse, out_grad=do, dq=dq, dk=dk, dv=dv, scale=base.SCALE)
    _times_out()
    again = base._run_cross(q, k, v, None, do)
    assert all(torch.equal(again[n], want[n]) for n in want)


@pytest.mark.parametrize("B,S", [(4, 1), (40, 4), (2, 300)])
def test_dropped_load_of_a_prefix(gpu, monkeypatch, B, S):
    import torch

    q, k, v, _ = base._inputs(B, S, 200, 8, 2, 81)
    pk, pv = base._inputs(1, 3000, 1, 2, 2, 82)[0][0], base._inputs(1, 3000, 1, 2, 2, 83)[0][0]
    out, lse = torch.empty_like(q), torch.empty(B, 8, S, device="cuda")
    kw = dict(q=q, prefix_k=pk, prefix_v=pv, k=k, v=v, out=out, lse=lse, scale=base.SCALE)
    with _dropped(monkeypatch, 0):
        base._rt().prefix_attn_fwd(**kw)
    _times_out()
    base._rt().prefix_attn_fwd(**kw)
    base._check_attention(q, k, v, [200] * B, dict(out=out, lse=lse), prefix=(pk, pv))
