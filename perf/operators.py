"""The workloads the conditioning operators are timed on.

Four operators that stand beside the block-sparse self-attention of a video
transformer: cross attention to an encoder's states (forward, and forward
with backward), attention of a batch over one shared prefix, and the per-head
RMSNorm of queries and keys with their position rotation (forward, and
forward with backward).  ``run`` computes each either in its plain form
(elementary torch operations in 32 bits) or, where ``own`` is true, with the
library's kernels.  ``exact`` restates each definition in 64 bits.

All operands are bf16 with a head dimension of 128; a batch's encoder states
are padded to one length and ``kv_lens`` holds each member's valid keys.
"""
import math
import os
import sys

import torch

own = False

D = 128
EPS = 1e-6
SCALE = D ** -0.5
ROPE_DIMS = (32, 48, 48)  # rotary channels of the t, h, w axes
THETA = 1e4


# ------------------------------------------------------------------- cases
def listed():
    """The listed cases; ``op`` names the operator, the rest its sizes."""
    return [
        # one query token of a guided pair against a short prompt: latency
        dict(name="cross one token", op="cross", batch=2, q_len=1, kv_len=77, heads=8, kv_heads=8, lens="ragged"),
        # a guided pair of 32x32x32 latent grids, prompt states padded to 512
        dict(name="cross guided pair", op="cross", batch=2, q_len=32768, kv_len=512, heads=40, kv_heads=40,
             lens="ragged"),
        # a 16x16x16 grid against the long states of a reference clip, grouped key/value heads
        dict(name="cross long states", op="cross", batch=1, q_len=4096, kv_len=16384, heads=40, kv_heads=8,
             lens="full"),
        # a small training step: odd sizes, grouped heads, one member without any prompt
        dict(name="cross train small", op="cross_train", batch=3, q_len=257, kv_len=77, heads=8, kv_heads=2,
             lens="empty"),
        # a 480x864 5 s clip (15,731 packed tokens, 56 heads) against its 332 text tokens
        dict(name="cross train clip", op="cross_train", batch=1, q_len=15731, kv_len=332, heads=56, kv_heads=56,
             lens="full"),
        # a batch of two with longer, ragged states: the largest training step
        dict(name="cross train long", op="cross_train", batch=2, q_len=16384, kv_len=1024, heads=40, kv_heads=40,
             lens="ragged"),
        # a few members, one token each, over a medium shared prefix: latency
        dict(name="prefix few tokens", op="prefix", batch=4, q_len=1, prefix_len=1000, kv_len=33, heads=8,
             kv_heads=2, lens="ragged"),
        # many members, one token each, over a prefix of 64k tokens: memory bandwidth
        dict(name="prefix many tokens", op="prefix", batch=32, q_len=1, prefix_len=65536, kv_len=512, heads=40,
             kv_heads=8, lens="ragged"),
        # four variants of a render over the 746 conditioning rows that they share
        dict(name="prefix four renders", op="prefix", batch=4, q_len=4096, prefix_len=746, kv_len=4096, heads=40,
             kv_heads=40, lens="full"),
        # one new token's queries and keys: latency
        dict(name="norm one token", op="norm", batch=2, q_len=1, kv_len=1, heads=8, kv_heads=2, k_rope=True),
        # a 5 s 1344x768 clip (31x48x84 grid) and its unrotated encoder keys: memory bandwidth
        dict(name="norm clip", op="norm", batch=1, q_len=124992, kv_len=512, heads=40, kv_heads=40, k_rope=False),
        # the same pass with its gradients, self-attention keys rotated too
        dict(name="norm train", op="norm_train", batch=1, q_len=32768, kv_len=32768, heads=40, kv_heads=40,
             k_rope=True),
    ]


def _spread(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the same ranges, at most the cost of the largest listed one of its operator."""
    op = rng.choice(["cross", "cross", "cross_train", "cross_train", "prefix", "prefix", "norm", "norm_train"])
    kv_heads = rng.choice([1, 2, 3, 5, 8, 14, 40])
    group = rng.choice([g for g in (1, 1, 1, 2, 4, 5, 8) if kv_heads * g <= 56])
    heads = kv_heads * group
    case = dict(op=op, batch=rng.choice([1, 2, 3, 4]), heads=heads, kv_heads=kv_heads)
    if op in ("norm", "norm_train"):
        q_len = _spread(rng, 1, 124992 if op == "norm" else 32768)
        while case["batch"] * q_len * heads > 124992 * 40:
            q_len = max(1, q_len // 2)
        kv_len = q_len if rng.random() < 0.5 else _spread(rng, 1, 1024)
        if op == "norm_train":
            while case["batch"] * (q_len * heads + kv_len * kv_heads) > 2 * 32768 * 40:
                q_len, kv_len = max(1, q_len // 2), max(1, kv_len // 2)
        return dict(case, q_len=q_len, kv_len=kv_len, k_rope=rng.random() < 0.5)
    case["lens"] = rng.choice(["full", "ragged", "ragged", "empty"])
    if op == "prefix":
        if rng.random() < 0.5:  # single tokens over a long prefix
            case["batch"] = rng.choice([1, 2, 5, 8, 16, 32])
            case.update(q_len=rng.choice([1, 1, 1, 2, 4]), prefix_len=_spread(rng, 128, 65536),
                        kv_len=_spread(rng, 1, 512))
        else:
            case.update(q_len=_spread(rng, 16, 4096), prefix_len=_spread(rng, 16, 4096), kv_len=_spread(rng, 1, 4096))
        keys = lambda: case["prefix_len"] + case["kv_len"]  # noqa: E731
        while case["batch"] * case["q_len"] * heads * keys() > 4 * 4096 * 40 * 4842:
            case["q_len"] = max(1, case["q_len"] // 2)
        return case
    case.update(q_len=_spread(rng, 1, 32768), kv_len=_spread(rng, 1, 16384 if op == "cross" else 4096))
    most = 2 * 32768 * 40 * 512 if op == "cross" else 2 * 16384 * 40 * 1024
    while case["batch"] * case["q_len"] * heads * case["kv_len"] > most:
        case["q_len"] = max(1, case["q_len"] // 2)
    return case


def _lens(case):
    """Valid keys of each member: all, falling from member to member, or none for the last."""
    b, n = case["batch"], case["kv_len"]
    if case["lens"] == "full":
        return [n] * b
    lens = [max(1, n - (3 * n * i) // (4 * b)) for i in range(b)]
    if case["lens"] == "empty":
        lens[-1] = 0
    return lens


# ------------------------------------------------------------------ inputs
def _table(grid):
    """bf16 [tokens, 64, 4] rotation table (c, -s, s, c) of a raster of t x h x w positions."""
    axes = [torch.arange(n, device="cuda", dtype=torch.float64) for n in grid]
    pos = torch.stack([p.reshape(-1) for p in torch.meshgrid(*axes, indexing="ij")], 1)
    angles = torch.cat([pos[:, a:a + 1] * THETA ** (-torch.arange(0, n, 2, device="cuda", dtype=torch.float64) / n)
                        for a, n in enumerate(ROPE_DIMS)], 1)
    c, s = angles.cos(), angles.sin()
    return torch.stack([c, -s, s, c], -1).to(torch.bfloat16).contiguous()


def _tokens_table(n):
    """The table of the first n tokens of a video raster 16 wide and 16 high."""
    return _table((-(-n // 256), 16, 16))[:n].contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    b, hq, hk, sq, sk = case["batch"], case["heads"], case["kv_heads"], case["q_len"], case["kv_len"]

    def normal(*shape, std=1.0, mean=0.0, dtype=torch.bfloat16):
        return torch.empty(shape, dtype=dtype, device="cuda").normal_(mean, std, generator=g)

    def like(*shape, dtype=torch.bfloat16):
        return torch.empty(shape, dtype=dtype, device="cuda")

    st = dict(case=case, q=normal(b, sq, hq, D), k=normal(b, sk, hk, D))
    if case["op"] in ("norm", "norm_train"):
        st.update(q_norm=normal(D, std=0.02, mean=1.0), k_norm=normal(D, std=0.02, mean=1.0),
                  q_rope=_tokens_table(sq), k_rope=_tokens_table(sk) if case["k_rope"] else None,
                  q_out=like(b, sq, hq, D), k_out=like(b, sk, hk, D))
        if case["op"] == "norm_train":
            st.update(q_grad=normal(b, sq, hq, D), k_grad=normal(b, sk, hk, D), dq=like(b, sq, hq, D),
                      dk=like(b, sk, hk, D), dq_norm=like(D, dtype=torch.float32), dk_norm=like(D, dtype=torch.float32))
        return st
    st.update(v=normal(b, sk, hk, D), out=like(b, sq, hq, D), lse=like(b, hq, sq, dtype=torch.float32),
              kv_lens=torch.tensor(_lens(case), dtype=torch.int32, device="cuda"))
    if case["op"] == "prefix":
        st.update(prefix_k=normal(case["prefix_len"], hk, D), prefix_v=normal(case["prefix_len"], hk, D))
    if case["op"] == "cross_train":
        st.update(out_grad=normal(b, sq, hq, D), dq=like(b, sq, hq, D), dk=like(b, sk, hk, D), dv=like(b, sk, hk, D))
    return st


# -------------------------------------------------------------- plain forms
def _heads_first(x, groups=1):
    """fp32 [batch, heads, tokens, D] of a [batch, tokens, heads, D] operand, key heads repeated for their group."""
    x = x.float().transpose(1, 2)
    return x.repeat_interleave(groups, 1) if groups > 1 else x


def _weights(q, k, mask):
    """Softmax weights [.., queries, keys] and their log-sum-exp; a row without keys has weights of 0 and -inf."""
    s = torch.matmul(q, k.transpose(-1, -2)).mul_(SCALE)
    s = s.masked_fill_(~mask, -math.inf)
    top = s.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    p = s.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    lse = torch.where(total > 0, total.log() + top, torch.full_like(total, -math.inf))
    return p.div_(total.clamp_min(1e-30)), lse.squeeze(-1)


def _valid(st):
    """[batch, 1, 1, keys]: the keys below each member's length."""
    return (torch.arange(st["k"].shape[1], device="cuda") < st["kv_lens"][:, None])[:, None, None, :]


def _plain_cross(st):
    groups = st["case"]["heads"] // st["case"]["kv_heads"]
    q, k, v = _heads_first(st["q"]), _heads_first(st["k"], groups), _heads_first(st["v"], groups)
    p, lse = _weights(q, k, _valid(st))
    out = torch.matmul(p, v)
    st["out"].copy_(out.transpose(1, 2))
    st["lse"].copy_(lse)
    return q, k, v, p


def _plain_cross_grads(st, q, k, v, p):
    groups = st["case"]["heads"] // st["case"]["kv_heads"]

    def shared(x):  # sum over the query heads of each key head
        b, h, s, d = x.shape
        return x.reshape(b, h // groups, groups, s, d).sum(2).transpose(1, 2)

    do = _heads_first(st["out_grad"])
    st["dv"].copy_(shared(torch.matmul(p.transpose(-1, -2), do)))
    dp = torch.matmul(do, v.transpose(-1, -2))
    ds = dp.sub_((p * dp).sum(-1, keepdim=True)).mul_(p).mul_(SCALE)
    st["dq"].copy_(torch.matmul(ds, k).transpose(1, 2))
    st["dk"].copy_(shared(torch.matmul(ds.transpose(-1, -2), q)))


def _plain_prefix(st):
    b, groups = st["case"]["batch"], st["case"]["heads"] // st["case"]["kv_heads"]
    k, v = (torch.cat([_heads_first(pre[None], groups).expand(b, -1, -1, -1), _heads_first(x, groups)], 2)
            for pre, x in ((st["prefix_k"], st["k"]), (st["prefix_v"], st["v"])))
    mask = _valid(st)
    mask = torch.cat([mask.new_ones(b, 1, 1, st["case"]["prefix_len"]), mask], -1)
    p, lse = _weights(_heads_first(st["q"]), k, mask)
    st["out"].copy_(torch.matmul(p, v).transpose(1, 2))
    st["lse"].copy_(lse)


def _rotate(x, table, back=False):
    """The 2x2 rotation of channel pairs (i, half + i) by table rows (t0, t1, t2, t3), or by their transpose."""
    if table is None:
        return x
    t, half = table.float()[None, :, None, :, :], table.shape[1]
    a, b = x[..., :half], x[..., half:2 * half]
    t1, t2 = (t[..., 2], t[..., 1]) if back else (t[..., 1], t[..., 2])
    return torch.cat([t[..., 0] * a + t1 * b, t2 * a + t[..., 3] * b, x[..., 2 * half:]], -1)


def _plain_norm(x, w, table, out):
    x = x.float()
    out.copy_(_rotate(x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float(), table))


def _plain_norm_grads(x, w, table, grad, dx, dw):
    x, g = x.float(), _rotate(grad.float(), table, back=True)
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    unit = x * r
    gw = g * w.float()
    dx.copy_(r * (gw - unit * (gw * unit).mean(-1, keepdim=True)))
    dw.copy_((g * unit).sum((0, 1, 2), dtype=torch.float64))


# --------------------------------------------------------------------- run
def _library():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    pkg = os.path.join(root, "minimax-h3-swift_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from h3attention import Runtime

    return Runtime.get(torch.cuda.current_device())


def run(st):
    op = st["case"]["op"]
    if op == "cross" or op == "cross_train":
        if own:
            rt = _library()
            rt.cross_attn_fwd(q=st["q"], k=st["k"], v=st["v"], out=st["out"], lse=st["lse"], kv_lens=st["kv_lens"],
                              scale=SCALE, layout="SHD")
        else:
            saved = _plain_cross(st)
        if op == "cross":
            return dict(out=st["out"], lse=st["lse"])
        if own:
            rt.cross_attn_bwd(q=st["q"], k=st["k"], v=st["v"], out=st["out"], lse=st["lse"], out_grad=st["out_grad"],
                              dq=st["dq"], dk=st["dk"], dv=st["dv"], kv_lens=st["kv_lens"], scale=SCALE, layout="SHD")
        else:
            _plain_cross_grads(st, *saved)
        return dict(out=st["out"], lse=st["lse"], dq=st["dq"], dk=st["dk"], dv=st["dv"])
    if op == "prefix":
        if own:
            _library().prefix_attn_fwd(q=st["q"], prefix_k=st["prefix_k"], prefix_v=st["prefix_v"], k=st["k"],
                                       v=st["v"], out=st["out"], lse=st["lse"], kv_lens=st["kv_lens"], scale=SCALE,
                                       layout="SHD")
        else:
            _plain_prefix(st)
        return dict(out=st["out"], lse=st["lse"])
    if own:
        rt = _library()
        rt.qk_norm_rope_fwd(q=st["q"], k=st["k"], q_out=st["q_out"], k_out=st["k_out"], q_norm=st["q_norm"],
                            k_norm=st["k_norm"], eps=EPS, q_rope=st["q_rope"], k_rope=st["k_rope"], layout="SHD")
    else:
        _plain_norm(st["q"], st["q_norm"], st["q_rope"], st["q_out"])
        _plain_norm(st["k"], st["k_norm"], st["k_rope"], st["k_out"])
    if op == "norm":
        return dict(q=st["q_out"], k=st["k_out"])
    if own:
        rt.qk_norm_rope_bwd(q=st["q"], k=st["k"], q_grad=st["q_grad"], k_grad=st["k_grad"], q_norm=st["q_norm"],
                            k_norm=st["k_norm"], dq=st["dq"], dk=st["dk"], dq_norm=st["dq_norm"],
                            dk_norm=st["dk_norm"], eps=EPS, q_rope=st["q_rope"], k_rope=st["k_rope"], layout="SHD")
    else:
        _plain_norm_grads(st["q"], st["q_norm"], st["q_rope"], st["q_grad"], st["dq"], st["dq_norm"])
        _plain_norm_grads(st["k"], st["k_norm"], st["k_rope"], st["k_grad"], st["dk"], st["dk_norm"])
    return dict(q=st["q_out"], k=st["k_out"], dq=st["dq"], dk=st["dk"], dq_norm=st["dq_norm"], dk_norm=st["dk_norm"])


def work(case):
    """Bytes and operations that one pass cannot do without."""
    b, hq, hk, sq, sk = case["batch"], case["heads"], case["kv_heads"], case["q_len"], case["kv_len"]
    rows = b * (sq * hq + sk * hk)
    if case["op"] in ("norm", "norm_train"):
        tables = 64 * 8 * (sq + (sk if case["k_rope"] else 0))
        if case["op"] == "norm":
            return {"bytes": rows * 512 + tables + 512, "flops": rows * 10 * D}
        return {"bytes": rows * 1024 + tables + 1536, "flops": rows * 30 * D}
    lens = _lens(case)
    keys = sum(lens)
    q_bytes, kv_bytes, lse = b * sq * hq * D * 2, keys * hk * D * 2, b * sq * hq * 4
    if case["op"] == "prefix":
        p = case["prefix_len"]
        return {"bytes": 2 * q_bytes + 2 * kv_bytes + 4 * p * hk * D + lse, "flops": 4 * hq * D * sq * (b * p + keys)}
    if case["op"] == "cross":
        return {"bytes": 2 * q_bytes + 2 * kv_bytes + lse, "flops": 4 * hq * D * sq * keys}
    grads = 2 * b * sk * hk * D * 2
    return {"bytes": 4 * q_bytes + 2 * kv_bytes + grads + lse, "flops": 14 * hq * D * sq * keys}


# ------------------------------------------------------------------- exact
def _exact_attention(case, q, k, v, do):
    """Output, log-sum-exp and, where ``do`` is given, the gradients of one member and key head in 64 bits:
    q, do [queries, group, D], k, v [keys, D]."""
    n, grp, _ = q.shape
    out, lse = torch.zeros_like(q), torch.full((n, grp), -math.inf, dtype=torch.float64, device=q.device)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    if k.shape[0]:
        step = max(1, (1 << 27) // (grp * k.shape[0]))
        for i in range(0, n, step):
            rows = q[i:i + step].reshape(-1, D)
            score = rows @ k.T * SCALE
            l_ = torch.logsumexp(score, 1)
            w = torch.exp(score - l_[:, None])
            o = w @ v
            out[i:i + step], lse[i:i + step] = o.view(-1, grp, D), l_.view(-1, grp)
            if do is not None:
                d = do[i:i + step].reshape(-1, D)
                dscore = w * (d @ v.T - (d * o).sum(1, keepdim=True)) * SCALE
                dq[i:i + step] = (dscore @ k).view(-1, grp, D)
                dk += dscore.T @ rows
                dv += w.T @ d
    return out, lse, dq, dk, dv


def _exact_norm(x, w, table, grad):
    """The normalised and rotated rows and, where ``grad`` is given, the gradients of x and w, in 64 bits."""
    x, w = x.double(), w.double()
    rms = torch.sqrt((x * x).sum(-1, keepdim=True) / D + EPS)
    y = x / rms * w
    half = 0 if table is None else table.shape[1]
    lo, hi, rest = slice(0, half), slice(half, 2 * half), slice(2 * half, D)
    m = torch.zeros(x.shape[1], 1, 0, 4, dtype=torch.float64, device=x.device) if table is None else table.double()[:, None]
    out = torch.empty_like(y)
    out[..., lo] = m[..., 0] * y[..., lo] + m[..., 1] * y[..., hi]
    out[..., hi] = m[..., 2] * y[..., lo] + m[..., 3] * y[..., hi]
    out[..., rest] = y[..., rest]
    if grad is None:
        return out, None, None
    grad = grad.double()
    g = torch.empty_like(y)
    g[..., lo] = m[..., 0] * grad[..., lo] + m[..., 2] * grad[..., hi]
    g[..., hi] = m[..., 1] * grad[..., lo] + m[..., 3] * grad[..., hi]
    g[..., rest] = grad[..., rest]
    dw = (g * x / rms).sum((0, 1, 2))
    gw = g * w
    return out, gw / rms - x * (gw * x).sum(-1, keepdim=True) / (D * rms ** 3), dw


def exact(case, seed):
    """What ``run`` returns, from the definitions in 64 bits."""
    st = prepare(case, seed)
    if case["op"] in ("norm", "norm_train"):
        train = case["op"] == "norm_train"
        res = {}
        for n in "qk":
            y, dx, dw = _exact_norm(st[n], st[n + "_norm"], st[n + "_rope"], st[n + "_grad"] if train else None)
            res[n] = y
            if train:
                res["d" + n], res["d" + n + "_norm"] = dx, dw
        order = ("q", "k", "dq", "dk", "dq_norm", "dk_norm") if train else ("q", "k")
        return {n: res[n] for n in order}
    train, hk = case["op"] == "cross_train", case["kv_heads"]
    grp = case["heads"] // hk
    res = {n: torch.zeros(st[n].shape, dtype=torch.float64, device="cuda")
           for n in (("out", "lse", "dq", "dk", "dv") if train else ("out", "lse"))}
    for b, n in enumerate(_lens(case)):
        for h in range(hk):
            mine = slice(h * grp, (h + 1) * grp)
            k, v = st["k"][b, :n, h].double(), st["v"][b, :n, h].double()
            if case["op"] == "prefix":
                k = torch.cat([st["prefix_k"][:, h].double(), k])
                v = torch.cat([st["prefix_v"][:, h].double(), v])
            do = st["out_grad"][b, :, mine].double() if train else None
            o, lse, dq, dk, dv = _exact_attention(case, st["q"][b, :, mine].double(), k, v, do)
            res["out"][b, :, mine], res["lse"][b, mine] = o, lse.T
            if train:
                res["dq"][b, :, mine], res["dk"][b, :n, h], res["dv"][b, :n, h] = dq, dk, dv
    return res
