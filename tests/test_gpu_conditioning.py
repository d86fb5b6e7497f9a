"""Cross attention and its gradient, attention over a shared prefix, and the
q/k norm with rotation against plain restatements in 64 bits (B200 only).

Tolerances, per element, from the roundings the kernels make (a bf16 rounding
is off by at most u = 2^-8 of the value):

* out = P v: u |out| for the result and u P|v| for the weights, which enter
  the product in bf16.
* dv = P^T do: likewise u |dv| + u P^T|do|.
* delta = do.out takes the rounded out, so it is off by at most
  e = sum |do| (u |out| + u P|v|); dS = P (dp - delta) by P e, and by u |dS|
  as it enters its products in bf16: dq: u |dq| + scale (u |dS| + P e) |k|,
  dk likewise with |q|.
* Up to 128 keys delta is sum(P dP) / sum(P) in fp32 instead, off by the
  shares of fp32 below: 2 c each for the weights and the products, of the sum
  of magnitudes sum P |do||v|.
* fp32: a logit is a sum of 128 products, off by at most 2^-23 of the sum of
  their magnitudes at each addition: c = 2^-16 max(scale sum |q k|), and a
  weight by that share (2^-20 more for exp2, log2 and the sums).  All terms
  above get that share of the sums of magnitudes on top.
* norm: u |y| and 2^-20 of the magnitudes that enter; the weights' gradients
  2^-24 n of the sum of magnitudes over their n rows.
"""
import math

import pytest

pytestmark = pytest.mark.gpu

D, U, SCALE = 128, 2.0 ** -8, 128 ** -0.5


def _rt():
    from h3attention import Runtime

    return Runtime.get(0)


def _normal(gen, *shape, mean=0.0, std=1.0):
    import torch

    return torch.empty(shape, device="cuda").normal_(mean, std, generator=gen).to(torch.bfloat16)


def _gen(seed):
    import torch

    return torch.Generator(device="cuda").manual_seed(seed)


def _assert_within(name, got, want, tol):
    import torch

    got = got.double()
    assert torch.isfinite(got).all(), f"{name}: not finite"
    worst = ((got - want).abs() - tol).max().item() if got.numel() else -1.0
    assert worst <= 0, f"{name}: {worst} over the tolerance (max error {(got - want).abs().max().item()})"


def _attention(q, k, v, scale, do=None, one_block=False):
    """One member in 64 bits: q, do [S, H, D], k, v [N, H, D] (heads already
    repeated).  Values and tolerances, by name."""
    import torch

    q, k, v = (x.double().transpose(0, 1) for x in (q, k, v))
    val, tol = {}, {}
    if k.shape[1] == 0:
        zero = torch.zeros_like(q)
        val["out"], val["lse"] = zero, torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
        tol["out"], tol["lse"] = zero, torch.zeros_like(val["lse"])
        if do is not None:
            val["dq"], val["dk"], val["dv"] = zero, torch.zeros_like(k), torch.zeros_like(v)
            tol.update({n: val[n] for n in ("dq", "dk", "dv")})
    else:
        s = q @ k.transpose(1, 2) * scale
        c = 2.0 ** -20 + 2.0 ** -16 * (q.abs() @ k.abs().transpose(1, 2) * scale).max().item() if q.numel() else 0.0
        lse = torch.logsumexp(s, 2)
        p = torch.exp(s - lse[..., None])
        out, mag = p @ v, p @ v.abs()
        val["out"], val["lse"] = out, lse
        tol["out"], tol["lse"] = U * out.abs() + (U + 2 * c) * mag + 1e-30, c + 2.0 ** -22 * lse.abs()
        if do is not None:
            g = do.double().transpose(0, 1)
            dp, delta = g @ v.transpose(1, 2), (g * out).sum(-1, keepdim=True)
            ds = p * (dp - delta)
            e = (g.abs() * tol["out"]).sum(-1, keepdim=True)
            if one_block:
                e = 4 * c * (p * (g.abs() @ v.abs().transpose(1, 2))).sum(-1, keepdim=True)
            eds = (U + 2 * c) * ds.abs() + p * (e + 2 * c * (g.abs() @ v.abs().transpose(1, 2) + delta.abs()))
            val["dv"], val["dq"], val["dk"] = p.transpose(1, 2) @ g, scale * ds @ k, scale * ds.transpose(1, 2) @ q
            tol["dv"] = U * val["dv"].abs() + (U + 2 * c) * p.transpose(1, 2) @ g.abs() + 1e-30
            tol["dq"] = U * val["dq"].abs() + scale * eds @ k.abs() + 1e-30
            tol["dk"] = U * val["dk"].abs() + scale * eds.transpose(1, 2) @ q.abs() + 1e-30
    return val, tol


def _check_attention(q, k, v, lens, got, do=None, prefix=None, scale=SCALE, one_block=False):
    """Compares got (out, lse and gradients, [B, S, H, D] and [B, H, S]) member by member."""
    import torch

    group = q.shape[2] // k.shape[2]
    for b, n in enumerate(lens):
        kk, vv = k[b, :n], v[b, :n]
        if prefix is not None:
            kk, vv = torch.cat([prefix[0], kk]), torch.cat([prefix[1], vv])
        kk, vv = kk.repeat_interleave(group, 1), vv.repeat_interleave(group, 1)
        val, tol = _attention(q[b], kk, vv, scale, None if do is None else do[b], one_block)
        _assert_within(f"out[{b}]", got["out"][b].transpose(0, 1), val["out"], tol["out"])
        if got.get("lse") is not None:
            if kk.shape[0] == 0:
                assert (got["lse"][b] == -math.inf).all()
            else:
                _assert_within(f"lse[{b}]", got["lse"][b], val["lse"], tol["lse"])
        if do is None:
            continue
        _assert_within(f"dq[{b}]", got["dq"][b].transpose(0, 1), val["dq"], tol["dq"])
        for name in ("dk", "dv"):
            mine = got[name][b].transpose(0, 1)
            assert (mine[:, n:] == 0).all(), f"{name}[{b}]: rows past the length are not 0"
            # the members of a group are summed in fp32 and rounded once: the tolerances add up
            w, t = (x.unflatten(0, (x.shape[0] // group, group)).sum(1) for x in (val[name], tol[name]))
            _assert_within(f"{name}[{b}]", mine[:, :n], w, t)


def _inputs(B, S, N, H, Hk, seed, pad=None, lens=None, std=1.0):
    g = _gen(seed)
    q, k, v, do = (_normal(g, B, s, h, D, std=std if i < 2 else 1.0)
                   for i, (s, h) in enumerate(((S, H), (N, Hk), (N, Hk), (S, H))))
    if pad is not None:
        for b, n in enumerate(lens):
            k[b, n:], v[b, n:] = pad, pad
    return q, k, v, do


def _lens_tensor(lens):
    import torch

    return torch.tensor(lens, dtype=torch.int32, device="cuda")


def _run_cross(q, k, v, lens=None, do=None, scale=SCALE, layout="SHD", stream=None):
    import torch

    rt = _rt()
    B, S, H, _ = q.shape
    lt = None if lens is None else _lens_tensor(lens)
    as_given = (lambda x: x) if layout == "SHD" else (lambda x: x.transpose(1, 2).contiguous())
    back = (lambda x: x) if layout == "SHD" else (lambda x: x.transpose(1, 2))
    q, k, v = as_given(q), as_given(k), as_given(v)
    out = torch.full_like(q, 7.0)
    lse = torch.full((B, H, S), 7.0, device="cuda")
    rt.cross_attn_fwd(q=q, k=k, v=v, out=out, lse=lse, kv_lens=lt, scale=scale, layout=layout, stream=stream)
    got = dict(out=back(out), lse=lse)
    if do is not None:
        do = as_given(do)
        dq, dk, dv = (torch.full(x.shape, 7.0, dtype=torch.bfloat16, device="cuda") for x in (q, k, v))
        rt.cross_attn_bwd(q=q, k=k, v=v, out=out, lse=lse, out_grad=do, dq=dq, dk=dk, dv=dv, kv_lens=lt, scale=scale,
                          layout=layout, stream=stream)
        got.update(dq=back(dq), dk=back(dk), dv=back(dv))
    return got


# (batch, q_len, kv_len, heads, kv_heads, lens)
CROSS = [
    (1, 1, 1, 1, 1, None), (1, 1, 77, 8, 8, None), (2, 1, 129, 8, 2, [129, 3]), (3, 2, 40, 5, 1, [0, 40, 1]),
    (1, 5, 128, 2, 2, None), (2, 127, 127, 2, 1, [127, 64]), (1, 128, 256, 3, 3, None), (2, 129, 257, 4, 2, [200, 257]),
    (1, 255, 383, 2, 2, None), (2, 256, 33, 3, 1, [33, 0]), (3, 257, 77, 8, 2, [77, 58, 0]), (1, 300, 600, 2, 1, [513]),
    (1, 1000, 332, 4, 4, None), (2, 515, 1024, 6, 2, [1024, 385]), (1, 64, 3001, 8, 2, None), (1, 16, 5000, 3, 3, [4999]),
    (70, 3, 20, 1, 1, [i % 21 for i in range(70)]), (1, 700, 2048, 1, 1, None),
    # several units and cut key tiles a CTA
    (2, 2500, 400, 10, 5, [400, 200]), (1, 4000, 332, 14, 14, None), (300, 2, 70, 4, 4, [i % 71 for i in range(300)]),
    (40, 40, 300, 8, 2, [300 - 7 * i for i in range(40)]),
]


@pytest.mark.parametrize("B,S,N,H,Hk,lens", CROSS, ids=["-".join(map(str, c[:5])) for c in CROSS])
def test_cross_matches_64_bits(gpu, B, S, N, H, Hk, lens):
    full = lens or [N] * B
    q, k, v, do = _inputs(B, S, N, H, Hk, 1, pad=float("nan"), lens=full)
    _check_attention(q, k, v, full, _run_cross(q, k, v, lens, do), do)


@pytest.mark.parametrize("pad", [float("nan"), float("inf"), -float("inf"), -3.3895e38])
def test_cross_padding_is_never_used(gpu, pad):
    lens = [130, 5, 0, 300]
    q, k, v, do = _inputs(4, 140, 300, 4, 2, 2, pad=pad, lens=lens)
    _check_attention(q, k, v, lens, _run_cross(q, k, v, lens, do), do)


def test_cross_lengths_are_clamped(gpu):
    q, k, v, do = _inputs(3, 20, 50, 2, 2, 3)
    _check_attention(q, k, v, [50, 0, 50], _run_cross(q, k, v, [51, -4, 2 ** 31 - 1], do), do)


@pytest.mark.parametrize("S,N", [(200, 300), (3, 700)])
def test_cross_heads_first_layout(gpu, S, N):
    q, k, v, do = _inputs(2, S, N, 4, 2, 4)
    _check_attention(q, k, v, [N, 77], _run_cross(q, k, v, [N, 77], do, layout="HSD"), do)


@pytest.mark.parametrize("std", [3.0, 0.05])
def test_cross_sharp_and_flat_rows(gpu, std):
    """Logits of +-100 (one key takes a row) and next to none."""
    q, k, v, do = _inputs(1, 150, 500, 2, 2, 5, std=std)
    _check_attention(q, k, v, [500], _run_cross(q, k, v, None, do), do)


def test_cross_growing_scores(gpu):
    """Keys that grow from block to block move the running maximum in every block."""
    import torch

    q, k, v, do = _inputs(1, 130, 1000, 2, 2, 6)
    grow = torch.linspace(0.2, 6.0, 1000, device="cuda")[None, :, None, None]
    q = (q.abs() * 0.3).to(torch.bfloat16)
    k = (k.abs() * grow).to(torch.bfloat16)
    _check_attention(q, k, v, [1000], _run_cross(q, k, v, None, do), do)


def test_cross_strided_and_broadcast_operands(gpu):
    """q, k, v as slices of packed projections; one set of states for the whole batch and for all heads."""
    import torch

    g = _gen(7)
    B, S, N, H = 2, 70, 150, 4
    q = _normal(g, B, S, 3, H, D)[:, :, 1]
    kv = _normal(g, 1, N, 2, 1, 136)[..., :D]
    k, v = kv[:, :, 0].expand(B, N, H, D), kv[:, :, 1].expand(B, N, H, D)
    do = _normal(g, B, S, H, D).expand(B, S, H, D)
    assert k.stride(0) == 0 and k.stride(2) == 0
    _check_attention(q, k, v, [N, 100], _run_cross(q, k, v, [N, 100], do), do)


def test_cross_writes_only_its_rows(gpu):
    """Outputs inside larger buffers: everything around them stays."""
    import torch

    q, k, v, do = _inputs(2, 131, 77, 2, 2, 8)
    bufs = {n: torch.full((2, s + 9, 3, D), 5.0, dtype=torch.bfloat16, device="cuda")
            for n, s in (("out", 131), ("dq", 131), ("dk", 77), ("dv", 77))}
    view = {n: b[:, 4:-5, :2] for n, b in bufs.items()}
    lse = torch.empty(2, 2, 131, device="cuda")
    rt = _rt()
    rt.cross_attn_fwd(q=q, k=k, v=v, out=view["out"], lse=lse, scale=SCALE)
    rt.cross_attn_bwd(q=q, k=k, v=v, lse=lse, out_grad=do, scale=SCALE, **view)
    _check_attention(q, k, v, [77, 77], dict(view, lse=lse), do)
    for n, b in bufs.items():
        view[n].fill_(5.0)
        assert (b == 5.0).all(), n


def test_cross_without_queries_or_keys(gpu):
    import torch

    q, k, v, do = _inputs(2, 6, 0, 4, 2, 9)
    _check_attention(q, k, v, [0, 0], _run_cross(q, k, v, None, do), do)
    q, k, v, do = _inputs(2, 0, 130, 4, 2, 9)
    got = _run_cross(q, k, v, None, do)
    assert (got["dk"] == 0).all() and (got["dv"] == 0).all()
    q, k, v, do = _inputs(0, 5, 5, 4, 2, 9)
    _run_cross(q, k, v, None, do)


def test_cross_long_strides(gpu):
    """Token strides that put the last rows more than 2^31 elements from the first."""
    import torch

    S, pitch = 140, 1 << 24
    big = torch.empty((S - 1) * pitch + D, dtype=torch.bfloat16, device="cuda")
    at = lambda: big.as_strided((1, S, 1, D), (0, pitch, D, 1))  # noqa: E731
    q, k, v, do = _inputs(1, S, S, 1, 1, 10)
    for n, x in (("q", q), ("k", k), ("v", v)):
        at().copy_(x)
        got = _run_cross(at() if n == "q" else q, at() if n == "k" else k, at() if n == "v" else v, None, do)
        _check_attention(q, k, v, [S], got, do)


def test_cross_gradient_of_few_keys(gpu):
    """Where keys are few dS is a small difference; with one key it is 0."""
    lens = [1, 2, 3, 5, 64, 65, 128, 0]
    q, k, v, do = _inputs(len(lens), 150, 128, 4, 2, 13)
    _check_attention(q, k, v, lens, _run_cross(q, k, v, lens, do), do, one_block=True)


def test_cross_is_deterministic(gpu):
    import torch

    q, k, v, do = _inputs(2, 900, 500, 6, 2, 11)
    a, b = _run_cross(q, k, v, [500, 300], do), _run_cross(q, k, v, [500, 300], do)
    assert all(torch.equal(a[n], b[n]) for n in a)


def test_cross_gradient_against_differences(gpu):
    """The gradient's product with a direction against a central difference of
    the plain loss in 64 bits: a second statement of the formula."""
    import torch

    q, k, v, do = _inputs(1, 40, 60, 2, 1, 12)
    got = _run_cross(q, k, v, None, do)

    def loss(q, k, v):
        s = torch.einsum("bshd,bnhd->bhsn", q, k.repeat_interleave(2, 2)) * SCALE
        return (torch.einsum("bhsn,bnhd->bshd", s.softmax(-1), v.repeat_interleave(2, 2)) * do.double()).sum()

    x = [t.double() for t in (q, k, v)]
    for i, n in enumerate(("dq", "dk", "dv")):
        d = torch.randn_like(x[i])
        h = 1e-4
        up, down = ([t + s * h * d if j == i else t for j, t in enumerate(x)] for s in (1, -1))
        want = ((loss(*up) - loss(*down)) / (2 * h)).item()
        have = (got[n].double() * d).sum().item()
        # every element is off by a few roundings (u = 2^-8) of its own size, with signs that do not agree
        assert abs(have - want) <= 8 * U * (got[n].double() * d).norm().item() + 1e-4 * abs(want), n


# ------------------------------------------------------------ shared prefix
# (batch, q_len, prefix, kv_len, heads, kv_heads, lens)
PREFIX = [
    (1, 1, 1, 0, 1, 1, None), (4, 1, 1000, 33, 8, 2, [33, 1, 0, 20]), (2, 1, 128, 128, 4, 4, None),
    (5, 2, 300, 7, 10, 2, [0, 1, 2, 3, 7]), (32, 1, 2000, 100, 5, 1, [i * 3 for i in range(32)]),
    (2, 1, 0, 50, 4, 2, [50, 0]), (3, 130, 200, 300, 2, 1, [300, 0, 129]), (2, 300, 77, 256, 4, 4, None),
    (40, 4, 700, 10, 8, 2, None), (2, 260, 640, 0, 2, 2, None), (1, 33, 4100, 65, 6, 3, None),
    (1, 520, 128, 1500, 2, 2, None),
]


@pytest.mark.parametrize("B,S,P,N,H,Hk,lens", PREFIX, ids=["-".join(map(str, c[:6])) for c in PREFIX])
def test_prefix_matches_64_bits(gpu, B, S, P, N, H, Hk, lens):
    import torch

    full = lens or [N] * B
    q, k, v, _ = _inputs(B, S, N, H, Hk, 20, pad=float("nan"), lens=full)
    pk, pv, _, _ = _inputs(1, P, 1, Hk, Hk, 21)[0][0], _inputs(1, P, 1, Hk, Hk, 22)[0][0], 0, 0
    out, lse = torch.full_like(q, 7.0), torch.full((B, H, S), 7.0, device="cuda")
    _rt().prefix_attn_fwd(q=q, prefix_k=pk, prefix_v=pv, k=k, v=v, out=out, lse=lse,
                          kv_lens=None if lens is None else _lens_tensor(lens), scale=SCALE)
    _check_attention(q, k, v, full, dict(out=out, lse=lse), prefix=(pk, pv))


@pytest.mark.parametrize("S", [1, 200])
def test_prefix_heads_first_without_lse(gpu, S):
    import torch

    q, k, v, _ = _inputs(3, S, 90, 4, 2, 23)
    pk, pv = _inputs(1, 500, 1, 2, 2, 24)[0][0], _inputs(1, 500, 1, 2, 2, 25)[0][0]
    out = torch.empty(3, 4, S, D, dtype=torch.bfloat16, device="cuda")
    hf = lambda x: x.transpose(-3, -2).contiguous()  # noqa: E731
    _rt().prefix_attn_fwd(q=hf(q), prefix_k=hf(pk), prefix_v=hf(pv), k=hf(k), v=hf(v), out=out, scale=SCALE,
                          layout="HSD")
    _check_attention(q, k, v, [90] * 3, dict(out=out.transpose(1, 2)), prefix=(pk, pv))


# ------------------------------------------------------------------ q/k norm
def _rope(tokens, half, seed, batch=None):
    """Tables need not hold rotations: any 2x2 entries are turned with."""
    shape = (tokens, half, 4) if batch is None else (batch, tokens, half, 4)
    return _normal(_gen(seed), *shape)


def _norm_reference(x, w, table, eps, grad):
    import torch

    x, w, g = x.double(), w.double(), grad.double()
    r = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    unit = x * r
    n = unit * w
    val, tol = {}, {}
    y, ymag, gr, gmag = n.clone(), n.abs(), g.clone(), g.abs()
    if table is not None:
        t = table.double()
        t = (t[None] if t.dim() == 3 else t)[:, :, None]
        h = t.shape[-2]
        a, b, ga, gb = n[..., :h], n[..., h:2 * h], g[..., :h], g[..., h:2 * h]
        y[..., :h], y[..., h:2 * h] = t[..., 0] * a + t[..., 1] * b, t[..., 2] * a + t[..., 3] * b
        gr[..., :h], gr[..., h:2 * h] = t[..., 0] * ga + t[..., 2] * gb, t[..., 1] * ga + t[..., 3] * gb
        t = t.abs()
        a, b, ga, gb = a.abs(), b.abs(), ga.abs(), gb.abs()
        ymag, gmag = ymag.clone(), gmag.clone()
        ymag[..., :h], ymag[..., h:2 * h] = t[..., 0] * a + t[..., 1] * b, t[..., 2] * a + t[..., 3] * b
        gmag[..., :h], gmag[..., h:2 * h] = t[..., 0] * ga + t[..., 2] * gb, t[..., 1] * ga + t[..., 3] * gb
    val["y"], tol["y"] = y, U * y.abs() + 2.0 ** -20 * ymag + 1e-38
    gw, gwmag = gr * w, gmag * w.abs()
    dx = r * (gw - unit * (gw * unit).mean(-1, keepdim=True))
    mag = r * (gwmag + unit.abs() * (gwmag * unit.abs()).mean(-1, keepdim=True))
    val["dx"], tol["dx"] = dx, U * dx.abs() + 2.0 ** -17 * mag + 1e-38
    rows = x.numel() // D
    val["dw"] = (gr * unit).sum((0, 1, 2))
    tol["dw"] = 2.0 ** -24 * (rows + 16) * (gmag * unit.abs()).sum((0, 1, 2)) + 1e-38
    return val, tol


# (batch, q_len, k_len, heads, kv_heads, q half, k half, tables for each member)
NORM = [
    (1, 1, 1, 1, 1, 64, 64, False), (2, 1, 1, 8, 2, 64, 64, False), (2, 33, 7, 5, 1, 64, None, False),
    (1, 100, 50, 3, 3, 48, 64, False), (3, 17, 20, 4, 2, None, 33, True), (2, 9, 40, 2, 1, 1, 8, True),
    (1, 1000, 77, 40, 8, 46, None, False), (1, 0, 5, 2, 1, 64, 64, False), (2, 5, 0, 2, 1, None, None, False),
    (0, 5, 5, 2, 1, 64, 64, False), (1, 700, 3, 14, 14, 64, 64, True),
    # runs of 2, 4 and 8 rows a group that end inside tokens, members and the operand
    (3, 6001, 600, 5, 1, 64, 40, False), (20001, 1, 2, 1, 1, 64, 64, True), (2, 40001, 3, 1, 1, 48, None, False),
    (2, 9001, 5003, 5, 3, 33, None, False),
]


@pytest.mark.parametrize("B,S,N,H,Hk,hq,hk,each", NORM, ids=["-".join(map(str, c)) for c in NORM])
@pytest.mark.parametrize("layout", ["SHD", "HSD"])
def test_norm_matches_64_bits(gpu, B, S, N, H, Hk, hq, hk, each, layout):
    import torch

    g = _gen(30)
    x = dict(q=_normal(g, B, S, H, D, std=2.0), k=_normal(g, B, N, Hk, D, std=0.01))
    grad = dict(q=_normal(g, B, S, H, D), k=_normal(g, B, N, Hk, D))
    w = dict(q=_normal(g, D, mean=1.0, std=0.5), k=_normal(g, D, mean=1.0, std=0.5))
    tab = dict(q=None if hq is None else _rope(S, hq, 31, B if each else None),
               k=None if hk is None else _rope(N, hk, 32, B if each else None))
    order = (lambda t: t) if layout == "SHD" else (lambda t: t.transpose(1, 2).contiguous())
    back = (lambda t: t) if layout == "SHD" else (lambda t: t.transpose(1, 2))
    rt = _rt()
    y = {n: torch.full_like(order(x[n]), 7.0) for n in x}
    kw = dict(q=order(x["q"]), k=order(x["k"]), q_norm=w["q"], k_norm=w["k"], eps=1e-5, q_rope=tab["q"],
              k_rope=tab["k"], layout=layout)
    rt.qk_norm_rope_fwd(q_out=y["q"], k_out=y["k"], **kw)
    d = {n: torch.full_like(order(x[n]), 7.0) for n in x}
    dw = {n: torch.full((D,), 7.0, device="cuda") for n in x}
    rt.qk_norm_rope_bwd(q_grad=order(grad["q"]), k_grad=order(grad["k"]), dq=d["q"], dk=d["k"], dq_norm=dw["q"],
                        dk_norm=dw["k"], **kw)
    for n in x:
        val, tol = _norm_reference(x[n], w[n], tab[n], 1e-5, grad[n])
        for name, got in (("y", back(y[n])), ("dx", back(d[n])), ("dw", dw[n])):
            _assert_within(n + " " + name, got, val[name], tol[name])


def test_norm_gradient_against_differences(gpu):
    """The gradients' products with a direction against central differences of
    the plain loss in 64 bits: a second statement of the formula."""
    import torch

    g = _gen(35)
    x, grad = _normal(g, 2, 30, 3, D), _normal(g, 2, 30, 3, D)
    w, tab = _normal(g, D, mean=1.0, std=0.5), _rope(30, 48, 36)
    dx, dk = torch.empty_like(x), torch.empty_like(x)
    dw, dwk = torch.empty(D, device="cuda"), torch.empty(D, device="cuda")
    _rt().qk_norm_rope_bwd(q=x, k=x, q_grad=grad, k_grad=grad, dq=dx, dk=dk, q_norm=w, k_norm=w, dq_norm=dw,
                           dk_norm=dwk, eps=1e-5, q_rope=tab)
    t = tab.double()[None, :, None]

    def loss(x, w):
        n = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5) * w
        a, b, rest = n[..., :48], n[..., 48:96], n[..., 96:]
        y = torch.cat([t[..., 0] * a + t[..., 1] * b, t[..., 2] * a + t[..., 3] * b, rest], -1)
        return (y * grad.double()).sum()

    at, h = [x.double(), w.double()], 1e-4
    for i, got in enumerate((dx, dw)):
        d = torch.randn_like(at[i])
        up, down = ([v + s * h * d if j == i else v for j, v in enumerate(at)] for s in (1, -1))
        want = ((loss(*up) - loss(*down)) / (2 * h)).item()
        have = (got.double() * d).sum().item()
        # every element is off by a rounding (u = 2^-8) of its own size, with signs that do not agree
        assert abs(have - want) <= 8 * U * (got.double() * d).norm().item() + 1e-4 * abs(want), i


def test_norm_in_place_and_strided(gpu):
    """Queries and keys as slices of one packed projection, normalised in place; gradients likewise."""
    import torch

    g = _gen(33)
    qkv, grads = _normal(g, 2, 50, 8, D), _normal(g, 2, 50, 8, D)
    w, tab = _normal(g, D, mean=1.0, std=0.1), _rope(50, 64, 34)
    ref_q = _norm_reference(qkv[:, :, :4], w, tab, 1e-6, grads[:, :, :4])
    ref_k = _norm_reference(qkv[:, :, 4:6], w, tab, 1e-6, grads[:, :, 4:6])
    work, gwork = qkv.clone(), grads.clone()
    dwq, dwk = torch.empty(D, device="cuda"), torch.empty(D, device="cuda")
    rt = _rt()
    rt.qk_norm_rope_bwd(q=work[:, :, :4], k=work[:, :, 4:6], q_grad=gwork[:, :, :4], k_grad=gwork[:, :, 4:6],
                        dq=gwork[:, :, :4], dk=gwork[:, :, 4:6], q_norm=w, k_norm=w, dq_norm=dwq, dk_norm=dwk,
                        q_rope=tab, k_rope=tab)
    rt.qk_norm_rope_fwd(q=work[:, :, :4], k=work[:, :, 4:6], q_out=work[:, :, :4], k_out=work[:, :, 4:6], q_norm=w,
                        k_norm=w, q_rope=tab, k_rope=tab)
    for (val, tol), at, dw in ((ref_q, slice(0, 4), dwq), (ref_k, slice(4, 6), dwk)):
        _assert_within("y", work[:, :, at], val["y"], tol["y"])
        _assert_within("dx", gwork[:, :, at], val["dx"], tol["dx"])
        _assert_within("dw", dw, val["dw"], tol["dw"])
    assert torch.equal(work[:, :, 6:], qkv[:, :, 6:]) and torch.equal(gwork[:, :, 6:], grads[:, :, 6:])


def test_norm_zero_rows(gpu):
    """All-zero rows: r = 1/sqrt(eps), no NaN, gradients finite."""
    import torch

    z = torch.zeros(1, 3, 2, D, dtype=torch.bfloat16, device="cuda")
    g, w = torch.ones_like(z), torch.ones(D, dtype=torch.bfloat16, device="cuda")
    y, dx, dk = torch.full_like(z, 7.0), torch.full_like(z, 7.0), torch.full_like(z, 7.0)
    dw, dwk = torch.empty(D, device="cuda"), torch.empty(D, device="cuda")
    _rt().qk_norm_rope_fwd(q=z, k=z, q_out=y, k_out=dk, q_norm=w, k_norm=w, eps=1e-6)
    _rt().qk_norm_rope_bwd(q=z, k=z, q_grad=g, k_grad=g, dq=dx, dk=dk, q_norm=w, k_norm=w, dq_norm=dw, dk_norm=dwk,
                           eps=1e-6)
    assert (y == 0).all() and (dw == 0).all()
    # r = 10^3, gradient of ones: 1000, within one rounding
    assert ((dx.double() - 1e3).abs() <= U * 1e3).all()


# ------------------------------------------------- streams, graphs, the whole
def _layer(st, rt, stream=None):
    """Norm and rotation of queries and encoder keys, cross attention, and the way back."""
    rt.qk_norm_rope_fwd(q=st["q"], k=st["k"], q_out=st["qn"], k_out=st["kn"], q_norm=st["wq"], k_norm=st["wk"],
                        q_rope=st["tab"], k_rope=None, stream=stream)
    rt.cross_attn_fwd(q=st["qn"], k=st["kn"], v=st["v"], out=st["out"], lse=st["lse"], kv_lens=st["lens"],
                      scale=SCALE, stream=stream)
    rt.cross_attn_bwd(q=st["qn"], k=st["kn"], v=st["v"], out=st["out"], lse=st["lse"], out_grad=st["do"],
                      dq=st["dqn"], dk=st["dkn"], dv=st["dv"], kv_lens=st["lens"], scale=SCALE, stream=stream)
    rt.qk_norm_rope_bwd(q=st["q"], k=st["k"], q_grad=st["dqn"], k_grad=st["dkn"], q_norm=st["wq"], k_norm=st["wk"],
                        dq=st["dq"], dk=st["dk"], dq_norm=st["dwq"], dk_norm=st["dwk"], q_rope=st["tab"], k_rope=None,
                        stream=stream)


RESULTS = ("out", "lse", "dv", "dq", "dk", "dwq", "dwk")


def _layer_state(seed, B=2, S=300, N=150, H=4, Hk=2):
    import torch

    g = _gen(seed)
    q, k, v, do = _inputs(B, S, N, H, Hk, seed)
    st = dict(q=q, k=k, v=v, do=do, wq=_normal(g, D, mean=1.0, std=0.1), wk=_normal(g, D, mean=1.0, std=0.1),
              tab=_rt().rope_table(torch.stack([torch.arange(S, device="cuda", dtype=torch.int32)] * 3, 1)),
              lens=_lens_tensor([N] + [N // 2] * (B - 1)), lse=torch.empty(B, H, S, device="cuda"),
              dwq=torch.empty(D, device="cuda"), dwk=torch.empty(D, device="cuda"))
    for n, like in (("qn", q), ("out", q), ("dqn", q), ("dq", q), ("kn", k), ("dkn", k), ("dk", k), ("dv", v)):
        st[n] = torch.empty_like(like)
    return st


@pytest.mark.parametrize("batch", [None, 2])
def test_cross_sdpa_is_the_call(gpu, batch):
    import torch

    from h3attention import cross_sdpa

    q, k, v, _ = _inputs(batch or 1, 140, 50, 4, 2, 60)
    lens = _lens_tensor([17] * (batch or 1))
    want = torch.empty_like(q)
    _rt().cross_attn_fwd(q=q, k=k, v=v, out=want, scale=SCALE, kv_lens=lens)
    if batch is None:
        q, k, v, want = q[0], k[0], v[0], want[0]
    assert torch.equal(cross_sdpa(q, k, v, D, kv_lens=lens), want.flatten(-2))


def test_layer_of_norm_and_cross_attention_has_the_gradients_of_the_whole(gpu):
    """The four calls in a row against torch.autograd over the plain layer in
    64 bits.  Each call is held to its own bound by the tests above; here the
    relative error of the whole is a few roundings: sqrt of the sum of squares
    of at most ten independent ones of u/sqrt(3) (norm output, weights, out,
    dS, gradients), below 4 u."""
    import torch

    st = _layer_state(40)
    _layer(st, _rt())
    x = {n: st[n].double().requires_grad_() for n in ("q", "k", "v", "wq", "wk")}

    def norm(t, w):
        return t / torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-6) * w

    qn, kn, t = norm(x["q"], x["wq"]), norm(x["k"], x["wk"]), st["tab"].double()[None, :, None]
    a, b = qn[..., :64], qn[..., 64:]
    qn = torch.cat([t[..., 0] * a + t[..., 1] * b, t[..., 2] * a + t[..., 3] * b], -1)
    s = torch.einsum("bshd,bnhd->bhsn", qn, kn.repeat_interleave(2, 2)) * SCALE
    mask = torch.arange(150, device="cuda") < st["lens"][:, None]
    s = s.masked_fill(~mask[:, None, None], -math.inf)
    out = torch.einsum("bhsn,bnhd->bshd", s.softmax(-1), x["v"].repeat_interleave(2, 2))
    out.backward(st["do"].double())
    want = dict(out=out, dv=x["v"].grad, dq=x["q"].grad, dk=x["k"].grad, dwq=x["wq"].grad, dwk=x["wk"].grad,
                lse=torch.logsumexp(s, -1))
    for n in RESULTS:
        rel = (st[n].double() - want[n]).norm() / want[n].norm()
        assert rel <= 4 * U, (n, rel.item())


def test_two_streams_at_once(gpu):
    import torch

    want = [_layer_state(s, S=2000) for s in (41, 42)]
    for st in want:
        _layer(st, _rt())
    got = [_layer_state(s, S=2000) for s in (41, 42)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        for st, s in zip(got, streams):
            _layer(st, _rt(), stream=s)
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(a[n], b[n]) for n in RESULTS)


def test_captured_graphs_replay_with_new_values(gpu):
    """Two captured layers, replayed in turn and after eager calls, on new input values."""
    import torch

    rt = _rt()
    sts = [_layer_state(43), _layer_state(44, B=1, S=70, N=300, H=2, Hk=1)]
    graphs = []
    for st in sts:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            _layer(st, rt)
        graphs.append(g)
    for seed in (45, 46):
        fresh = [_layer_state(seed), _layer_state(seed + 10, B=1, S=70, N=300, H=2, Hk=1)]
        for st, f in zip(sts, fresh):
            for n in ("q", "k", "v", "do", "wq", "wk"):
                st[n].copy_(f[n])
            _layer(f, rt)
        for g in graphs:
            g.replay()
        for g in reversed(graphs):
            g.replay()
        torch.cuda.synchronize()
        for st, f in zip(sts, fresh):
            assert all(torch.equal(st[n], f[n]) for n in RESULTS)


def test_captured_decode_over_a_prefix(gpu):
    import torch

    rt = _rt()
    q, k, v, _ = _inputs(4, 1, 40, 8, 2, 47)
    pk, pv = _inputs(1, 900, 1, 2, 2, 48)[0][0], _inputs(1, 900, 1, 2, 2, 49)[0][0]
    lens = _lens_tensor([40, 3, 0, 17])
    out, lse = torch.empty_like(q), torch.empty(4, 8, 1, device="cuda")
    kw = dict(q=q, prefix_k=pk, prefix_v=pv, k=k, v=v, kv_lens=lens, scale=SCALE)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        rt.prefix_attn_fwd(out=out, lse=lse, **kw)
    for step in range(3):  # the lengths grow on the device between replays
        g.replay()
        _check_attention(q, k, v, lens.tolist(), dict(out=out, lse=lse), prefix=(pk, pv))
        lens += 5
        lens.clamp_(max=40)
        q.copy_(_normal(_gen(50 + step), 4, 1, 8, D))


def test_refusals_leave_the_context_usable(gpu):
    import torch

    from h3attention import H3CError

    q, k, v, do = _inputs(1, 8, 8, 2, 2, 51)
    rt = _rt()
    with pytest.raises(H3CError, match="head_dim"):
        rt.cross_attn_fwd(q=q[..., :64], k=k[..., :64], v=v[..., :64], out=torch.empty_like(q)[..., :64], scale=SCALE)
    with pytest.raises(H3CError, match="scale"):
        rt.cross_attn_fwd(q=q, k=k, v=v, out=torch.empty_like(q), scale=-1.0)
    with pytest.raises(ValueError, match="out must have"):
        rt.cross_attn_fwd(q=q, k=k, v=v, out=torch.empty_like(q)[:, :4], scale=SCALE)
    with pytest.raises(ValueError, match="bfloat16"):
        rt.cross_attn_fwd(q=q.half(), k=k, v=v, out=torch.empty_like(q), scale=SCALE)
    with pytest.raises(ValueError, match="kv_lens"):
        rt.cross_attn_fwd(q=q, k=k, v=v, out=torch.empty_like(q), scale=SCALE, kv_lens=torch.tensor([8], device="cuda"))
    with pytest.raises(H3CError, match="overlaps itself"):
        rt.cross_attn_fwd(q=q, k=k, v=v, out=torch.empty_like(q)[:, :, :1].expand(1, 8, 2, D), scale=SCALE)
    with pytest.raises(ValueError, match="q_rope"):
        rt.qk_norm_rope_fwd(q=q, k=k, q_out=q, k_out=k, q_norm=q[0, 0, 0], k_norm=k[0, 0, 0], q_rope=_rope(7, 64, 1))
    _check_attention(q, k, v, [8], _run_cross(q, k, v, None, do), do)


def test_workspace_is_checked(gpu):
    """A workspace that is missing or too small is refused, whatever the size asked for."""
    import ctypes as C

    import torch

    from h3attention import _lib

    rt = _rt()
    q, k, v, do = _inputs(1, 300, 300, 2, 1, 52)
    out, lse = torch.empty_like(q), torch.empty(1, 2, 300, device="cuda")
    view = lambda x: _lib.BView(x.data_ptr(), x.stride(0), x.stride(1), x.stride(2))  # noqa: E731
    a, n = _lib.CrossArgs(), C.c_size_t()
    a.batch, a.q_len, a.kv_len, a.heads, a.kv_heads, a.head_dim, a.scale, a.lse = 1, 300, 300, 2, 1, 128, SCALE, lse.data_ptr()
    a.q, a.k, a.v, a.out, a.out_grad, a.dq, a.dk, a.dv = (
        view(x) for x in (q, k, v, out, do, torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)))
    L = _lib.load()
    assert L.h3c_cross_workspace_size(C.byref(a), _lib.H3C_OP_CROSS_BWD, C.byref(n), None, 0) == _lib.H3C_OK and n.value
    ws = torch.empty(n.value, dtype=torch.uint8, device="cuda")
    for ptr, size in ((None, n.value), (ws.data_ptr(), n.value - 1)):
        a.workspace, a.workspace_bytes = ptr, size
        assert L.h3c_cross_attn_bwd(rt.ctx, C.byref(a), None) == _lib.H3C_ERR_CAPACITY
    a.workspace, a.workspace_bytes = ws.data_ptr() + 128, n.value
    assert L.h3c_cross_attn_bwd(rt.ctx, C.byref(a), None) == _lib.H3C_ERR_UNSUPPORTED
