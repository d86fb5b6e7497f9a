"""Conditioning calls from several host threads at once (B200 only)."""
import ctypes as C
import threading

import pytest

import test_gpu_conditioning as base

pytestmark = pytest.mark.gpu


def test_refusals_from_several_threads_keep_their_own_reasons(gpu):
    """Threads that are refused at once, with reasons of different lengths, each
    read the whole of their own."""
    from h3attention import _lib

    rt, L = base._rt(), _lib.load()
    spoilt = [("scale", -1.0, b"scale must be positive"), ("head_dim", 64, b"head_dim must be 128"),
              ("reserved", 1, b"bad batch, lengths, heads or reserved"), ("heads", 3, b"heads must be a multiple of kv_heads")]
    wrong, go = [], threading.Barrier(len(spoilt))

    def refused(name, value, why):
        a = _lib.CrossArgs()
        a.batch, a.q_len, a.kv_len, a.heads, a.kv_heads, a.head_dim, a.scale = 1, 1, 1, 2, 2, 128, 1.0
        setattr(a, name, value)
        go.wait()
        for _ in range(20000):
            if L.h3c_cross_attn_fwd(rt.ctx, C.byref(a), None) == _lib.H3C_OK:
                wrong.append((name, "not refused"))
                return
            said = L.h3c_last_error(rt.ctx)
            if not said.startswith(b"h3c_cross_attn_fwd: " + why):
                wrong.append((name, said))
                return

    threads = [threading.Thread(target=refused, args=s) for s in spoilt]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong
    assert L.h3c_last_error(rt.ctx)  # this thread had no failure of its own: the context's last


def test_two_threads_at_once(gpu):
    """Two threads, each with its stream, make the calls of a layer."""
    import torch

    rt = base._rt()
    want = [base._layer_state(s, S=700) for s in (86, 87)]
    for st in want:
        base._layer(st, rt)
    got = [base._layer_state(s, S=700) for s in (86, 87)]
    torch.cuda.synchronize()
    failed = []

    def work(st):
        try:
            stream = torch.cuda.Stream()
            for _ in range(20):
                base._layer(st, rt, stream=stream)
            stream.synchronize()
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(st,)) for st in got]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    for a, b in zip(want, got):
        assert all(torch.equal(a[n], b[n]) for n in base.RESULTS)
