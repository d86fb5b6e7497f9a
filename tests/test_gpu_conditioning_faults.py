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


def test_a_failed_call_leaves_the_others_alone(gpu, monkeypatch):
    """Calls beside and behind one whose waits ran out, before anyone has read
    the status: right results, of the self-attention too; and the other way round."""
    import torch

    from h3attention import BlockList, H3CError, MaskSpec

    rt = base._rt()
    q, k, v, do = base._inputs(2, 2500, 400, 10, 5, 84)
    want = base._run_cross(q, k, v, [400, 200], do)
    lens = base._lens_tensor([400, 200])
    g = torch.cuda.CUDAGraph()
    replayed, lse = torch.empty_like(q), torch.empty(2, 10, 2500, device="cuda")
    with torch.cuda.graph(g):
        rt.cross_attn_fwd(q=q, k=k, v=v, out=replayed, lse=lse, kv_lens=lens, scale=base.SCALE)
    bl = BlockList.build(MaskSpec(seq_len=1024, frames=4, height=16, width=16, n_random=1, seed=3))
    x = base._inputs(1, 1024, 1024, 2, 2, 85)[:3]
    out = torch.empty_like(x[0][0])
    kw = dict(q=x[0][0], k=x[1][0], v=x[2][0], out=out, layout="SHD", scale=base.SCALE, blocks=bl.on(gpu))
    rt.attn_fwd_sync(**kw)
    attended = out.clone()

    def others_are_right():
        again = base._run_cross(q, k, v, [400, 200], do)
        assert all(torch.equal(again[n], want[n]) for n in again)
        replayed.fill_(7.0)
        g.replay()
        assert torch.equal(replayed, want["out"])

    fails, beside = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with _dropped(monkeypatch, 0), torch.cuda.stream(fails):
        base._run_cross(q, k, v, None)
    with torch.cuda.stream(beside):
        again = base._run_cross(q, k, v, [400, 200], do)
    torch.cuda.synchronize()
    assert all(torch.equal(again[n], want[n]) for n in again)
    others_are_right()
    out.fill_(7.0)
    rt.attn_fwd(**kw)
    torch.cuda.synchronize()
    assert torch.equal(out, attended)
    with pytest.raises(H3CError, match="^(?!.*h3c_attn_fwd).*h3c_cross_attn_fwd"):
        rt.device_status()
    rt.device_status()

    with _dropped(monkeypatch, 3):
        rt.attn_fwd(**kw)
    torch.cuda.synchronize()
    others_are_right()
    with pytest.raises(H3CError, match="^(?!.*h3c_cross_attn_fwd).*h3c_attn_fwd"):
        rt.device_status()
    rt.attn_fwd_sync(**kw)
    assert torch.equal(out, attended)
