"""Failure detection of the conditioning calls without a GPU fault: a barrier of
every block is made to wait for bytes that never come (a test hook read from the
environment), so that the bounded waits of one role, and with it of all, run
out after a short limit.  The context must report H3C_ERR_TIMEOUT and then give
right results again."""
import contextlib

import pytest

import test_gpu_conditioning as base

pytestmark = pytest.mark.gpu

# places in the forward kernels' barriers (two halves, rings of up to three)
Q_FULL, Q_EMPTY, KV_FULL, K_EMPTY, V_EMPTY = 0, 2, 4, 7, 10
S_FULL, P_HALF, P_FULL, O_FULL, O_EMPTY, ML_FULL = 13, 15, 17, 19, 21, 23
DENSE = [Q_EMPTY, KV_FULL, KV_FULL + 1, K_EMPTY, V_EMPTY + 1, S_FULL, S_FULL + 1, P_HALF, P_FULL + 1, O_FULL, O_FULL + 1,
         O_EMPTY, ML_FULL, ML_FULL + 1]
FOLDED = DENSE + [Q_FULL]


@contextlib.contextmanager
def _stalled(monkeypatch, barrier, limit_ns=20_000_000):
    with monkeypatch.context() as m:
        m.setenv("H3C_TEST_WAIT_LIMIT_NS", str(limit_ns))
        m.setenv("H3C_TEST_STALL_BARRIER", str(barrier))
        yield


def _times_out(barrier):
    import torch

    from h3attention import H3CError, _lib

    torch.cuda.synchronize()
    with pytest.raises(H3CError, match="bounded device wait") as e:
        base._rt().device_status()
        pytest.fail(f"barrier {barrier}: no wait ran out")
    assert e.value.status == _lib.H3C_ERR_TIMEOUT
    base._rt().device_status()  # cleared


# (batch, q_len, kv_len, heads, kv_heads, barriers); several units and key tiles a block, in every form of the kernels
CASES = [
    (40, 260, 300, 4, 4, DENSE), (24, 260, 700, 4, 4, DENSE),
    (16, 4, 3000, 8, 4, FOLDED), (12, 100, 1500, 8, 2, FOLDED),
]


@pytest.mark.parametrize("B,S,N,H,Hk,barriers", CASES, ids=["short", "dense", "single", "dual"])
def test_stalled_cross_attention(gpu, monkeypatch, B, S, N, H, Hk, barriers):
    import torch

    q, k, v, _ = base._inputs(B, S, N, H, Hk, 80)
    want = base._run_cross(q, k, v, None)
    for barrier in barriers:
        with _stalled(monkeypatch, barrier):
            base._run_cross(q, k, v, None)
        _times_out(barrier)
    again = base._run_cross(q, k, v, None)
    assert all(torch.equal(again[n], want[n]) for n in want)


@pytest.mark.parametrize("N,lens", [(100, None), (700, [700, 90] * 10)], ids=["one block", "several"])
def test_stalled_gradient(gpu, monkeypatch, N, lens):
    """Places 0 to 26 of dq's barriers and 0 to 17 of dk's and dv's, but for
    those that only an abort waits for (dq's 24)."""
    import torch

    q, k, v, do = base._inputs(20, 300, N, 8, 4, 80)
    want = base._run_cross(q, k, v, lens, do)
    lens = None if lens is None else base._lens_tensor(lens)
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    kw = dict(q=q, k=k, v=v, out=want["out"], lse=want["lse"], out_grad=do, dq=dq, dk=dk, dv=dv, kv_lens=lens,
              scale=base.SCALE)
    for barrier in range(27):
        if barrier != 24:
            with _stalled(monkeypatch, barrier):
                base._rt().cross_attn_bwd(**kw)
            _times_out(barrier)
    base._rt().cross_attn_bwd(**kw)
    assert all(torch.equal(x, want[n]) for n, x in (("dq", dq), ("dk", dk), ("dv", dv)))


@pytest.mark.parametrize("B,S", [(4, 1), (40, 4), (2, 300)])
def test_stalled_prefix(gpu, monkeypatch, B, S):
    import torch

    q, k, v, _ = base._inputs(B, S, 200, 8, 2, 81)
    pk, pv = base._inputs(1, 3000, 1, 2, 2, 82)[0][0], base._inputs(1, 3000, 1, 2, 2, 83)[0][0]
    out, lse = torch.empty_like(q), torch.empty(B, 8, S, device="cuda")
    kw = dict(q=q, prefix_k=pk, prefix_v=pv, k=k, v=v, out=out, lse=lse, scale=base.SCALE)
    for barrier in (KV_FULL, S_FULL, P_FULL, ML_FULL):
        with _stalled(monkeypatch, barrier):
            base._rt().prefix_attn_fwd(**kw)
        _times_out(barrier)
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
    with _stalled(monkeypatch, KV_FULL), torch.cuda.stream(fails):
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

    with monkeypatch.context() as m:
        m.setenv("H3C_TEST_WAIT_LIMIT_NS", "20000000")
        m.setenv("H3C_TEST_DROP_ITEM", "3")
        rt.attn_fwd(**kw)
    torch.cuda.synchronize()
    others_are_right()
    with pytest.raises(H3CError, match="^(?!.*h3c_cross_attn_fwd).*h3c_attn_fwd"):
        rt.device_status()
    rt.attn_fwd_sync(**kw)
    assert torch.equal(out, attended)
