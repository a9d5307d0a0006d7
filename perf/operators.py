"""Cases of the operators of a linear-attention student: what is timed and compared, and their plain forms.

Three operators and their directions, by a case's ``op``:

* ``linattn_fwd``, ``linattn_bwd``, ``linattn_step`` - linear attention with a decay for each head
  over a batch of sequences (``seq`` rows each, ``ragged``: of different lengths; ``states``: with
  the state of an earlier part going in and this part's going out), its gradients, and one token
  per sequence.
* ``join_fwd``, ``join_bwd`` - a block's output joined to the residual stream: norm, gate, residual
  scale and the next block's norm (``gate``: "none", "vector" or "sequence").
* ``distill`` - the loss of a student's logits against a teacher's top logits, with its gradient.

``run`` computes them with elementary torch operations in 32 bits, or, with ``own``, through
``jaxpp_amd.runtime``; ``exact`` from their definitions in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
DEV = "cuda"
EPS = 1e-6


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _lin(op, batch, seq, heads, kv, dim, dtype="bf16", ragged=False, states=True):
    c = dict(op=op, batch=batch, seq=seq, heads=heads, kv=kv, dim=dim, dtype=dtype)
    return c if op == "linattn_step" else dict(c, ragged=ragged, states=states)


def _join(op, batch, seq, cols, dtype="bf16", gate="vector", post=True):
    return dict(op=op, batch=batch, seq=seq, cols=cols, dtype=dtype, gate=gate, post=post)


def _distill(rows, vocab, k, dtype="bf16", temperature=1.0):
    return dict(op="distill", rows=rows, vocab=vocab, k=k, dtype=dtype, temperature=temperature)


def listed():
    return [
        # A short prompt of one user: a few dozen tokens, the smallest heads.  All latency.
        dict(_lin("linattn_fwd", 1, 77, 4, 4, 64), name="prompt, short"),
        # One long document through a layer of hidden 4096, state in and out.
        dict(_lin("linattn_fwd", 1, 16384, 32, 32, 128), name="prompt, long"),
        # A small float32 model's training step on sequences of different odd lengths.
        dict(_lin("linattn_bwd", 3, 333, 4, 4, 64, "f32", ragged=True, states=False), name="gradients, float32 ragged"),
        # The training microbatch of the repository's headline layer (hidden 4096, 4096 tokens,
        # 32 query heads on 8 shared ones), twice.
        dict(_lin("linattn_bwd", 2, 4096, 32, 8, 128, states=False), name="gradients, 2 x 4096 tokens"),
        # The next token of one user of a small float32 model, and of 64 users of a large one.
        dict(_lin("linattn_step", 1, 1, 8, 8, 64, "f32"), name="token, one user"),
        dict(_lin("linattn_step", 64, 1, 32, 32, 128), name="token, 64 users"),
        # The join between two blocks for one token, and for a large microbatch of hidden 4096.
        dict(_join("join_fwd", 1, 1, 4096), name="join, one token"),
        dict(_join("join_fwd", 4, 4096, 4096, gate="sequence"), name="join, 4 x 4096 tokens"),
        # Its gradients: a small float32 model with a gate for each sequence, and hidden 8192.
        dict(_join("join_bwd", 3, 333, 768, "f32", gate="sequence"), name="join gradients, float32"),
        dict(_join("join_bwd", 2, 4096, 8192), name="join gradients, hidden 8192"),
        # The loss of a handful of tokens over a vocabulary of odd size, float32 logits.
        dict(_distill(5, 50021, 10, "f32", temperature=2.0), name="distillation, 5 tokens"),
        # A microbatch of 4096 tokens over the vocabulary of a large model.  The largest.
        dict(_distill(4096, 128256, 64), name="distillation, 4096 tokens"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


MOST = {"linattn_fwd": 16384 * 32 * 128, "linattn_bwd": 8192 * 32 * 128, "linattn_step": 64 * 32 * 128 * 128,
        "join_fwd": 16384 * 4096, "join_bwd": 8192 * 8192, "distill": 4096 * 128256}


def draw(rng):
    while True:
        op = rng.choice(["linattn_fwd", "linattn_fwd", "linattn_bwd", "linattn_bwd", "linattn_step", "join_fwd",
                         "join_bwd", "distill", "distill"])
        dtype = "f32" if rng.random() < 0.25 else "bf16"
        small = 4 if dtype == "f32" else 1
        if op.startswith("linattn"):
            heads = _log_int(rng, 1, 64)
            group = rng.choice([1, 1, 1, 2, 4, 8])
            kv = max(1, heads // group)
            heads = kv * min(group, heads)
            dim = rng.choice([64, 128])
            if op == "linattn_step":
                c = _lin(op, _log_int(rng, 1, 256), 1, heads, kv, dim, dtype)
                size = c["batch"] * heads * dim * dim
            else:
                c = _lin(op, _log_int(rng, 1, 16), _log_int(rng, 1, 16384), heads, kv, dim, dtype,
                         rng.random() < 0.4, rng.random() < 0.5)
                size = c["batch"] * c["seq"] * heads * dim * small
        elif op.startswith("join"):
            c = _join(op, _log_int(rng, 1, 16), _log_int(rng, 1, 8192), 8 * _log_int(rng, 16, 1024), dtype,
                      rng.choice(["none", "vector", "sequence"]), rng.random() < 0.75)
            size = c["batch"] * c["seq"] * c["cols"] * small
        else:
            c = _distill(_log_int(rng, 1, 4096), _log_int(rng, 1000, 160000), _log_int(rng, 1, 128), dtype,
                         rng.choice([1.0, 1.0, 2.0, 0.5]))
            size = c["rows"] * c["vocab"] * small
        if size <= MOST[op] and 3072 not in c.values():
            return c


# ---------------------------------------------------------------------------
# what a user's program has in hand
# ---------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(int(seed) + 7919)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, generator=gen, device=DEV, dtype=torch.float32) * scale).to(dtype)

    def empty(*shape, dtype=dt):
        return torch.empty(*shape, device=DEV, dtype=dtype)

    s = dict(case)
    if case["op"].startswith("linattn"):
        b, t, h, hk, d = (case[n] for n in ("batch", "seq", "heads", "kv", "dim"))
        s["scale"] = d ** -0.5
        s["q"], s["k"], s["v"] = normal(b, t, h, d), normal(b, t, hk, d), normal(b, t, hk, d)
        # windows from 32 to 512 tokens over the heads, as such layers fix them
        window = torch.logspace(5, 9, h, base=2.0, device=DEV, dtype=torch.float64)
        s["decay"] = torch.log1p(-1.0 / window).to(torch.float32)
        # a state is a sum of about 1 / (1 - lambda^2) outer products
        reach = torch.rsqrt(-torch.expm1(2.0 * s["decay"]))[None, :, None, None]

        def state():
            return normal(b, h, d, d, dtype=torch.float32) * reach

        s["lens"] = None
        if case["op"] == "linattn_step":
            s["state_in"], s["state_out"], s["o"] = state(), empty(b, h, d, d, dtype=torch.float32), empty(b, t, h, d)
            return s
        if case["ragged"]:
            s["lens"] = torch.randint(t // 3, t + 1, (b,), generator=gen, device=DEV, dtype=torch.int32)
        s["state_in"] = state() if case["states"] else None
        backward = case["op"] == "linattn_bwd"
        if backward:
            s["d_o"] = normal(b, t, h, d)
            s["d_state_out"] = normal(b, h, d, d, dtype=torch.float32) if case["states"] else None
            s["dq"], s["dk"], s["dv"] = (torch.empty_like(s[n]) for n in "qkv")
        else:
            s["o"] = empty(b, t, h, d)
        s["state"] = empty(b, h, d, d, dtype=torch.float32) if case["states"] else None
        s["workspace"] = empty(_workspace(case, backward), dtype=torch.uint8)
    elif case["op"].startswith("join"):
        b, t, cols = case["batch"], case["seq"], case["cols"]
        rows, groups = b * t, {"none": 0, "vector": 1, "sequence": b}[case["gate"]]
        s["alpha"] = 0.9
        s["b"] = normal(rows, cols, scale=2.0)
        s["gamma_post"] = (1 + normal(cols, scale=0.1, dtype=torch.float32)).to(dt) if case["post"] else None
        s["gamma_pre"] = (1 + normal(cols, scale=0.1, dtype=torch.float32)).to(dt)
        s["gate"] = normal(groups, cols, scale=0.5) if groups else None
        s["gate_rows"] = rows // groups if groups else 0
        if case["op"] == "join_fwd":
            s["x"] = normal(rows, cols)
            s["h"], s["y"] = empty(rows, cols), empty(rows, cols)
            s["rstd_post"], s["rstd_pre"] = empty(rows, dtype=torch.float32), empty(rows, dtype=torch.float32)
        else:
            s["h"], s["dh"], s["dy"] = normal(rows, cols), normal(rows, cols, scale=0.1), normal(rows, cols, scale=0.1)
            s["rstd_post"] = torch.rsqrt(s["b"].float().square().mean(1) + EPS) if case["post"] else None
            s["rstd_pre"] = torch.rsqrt(s["h"].float().square().mean(1) + EPS)
            s["dx"], s["db"] = empty(rows, cols), empty(rows, cols)
            s["dgamma_pre"] = empty(cols, dtype=torch.float32)
            s["dgamma_post"] = empty(cols, dtype=torch.float32) if case["post"] else None
            s["dgate"] = empty(groups, cols, dtype=torch.float32) if groups else None
            # the gradient's sums over rows, one or a few lines for each group
            s["workspace"] = empty(2 * (max(groups, 1) + 512) * cols * 4, dtype=torch.uint8)
    else:
        rows, vocab, k = case["rows"], case["vocab"], case["k"]
        s["logits"] = normal(rows, vocab, scale=2.5)
        # distinct ids: places in `k` equal parts of the vocabulary
        k = min(k, vocab)
        part = vocab // k
        at = torch.randint(0, part, (rows, k), generator=gen, device=DEV)
        s["ids"] = (at + part * torch.arange(k, device=DEV)).to(torch.int32)
        top = normal(rows, k, scale=1.5, dtype=torch.float32) + 9.0
        s["teacher"] = torch.sort(top, dim=1, descending=True).values.contiguous()
        weight = (torch.rand(rows, generator=gen, device=DEV) < 0.9).float()     # prompts carry no loss
        weight[0] = 1.0
        s["weight"], s["scale"] = weight, 1.0 / rows
        s["row_loss"], s["loss"] = empty(rows, dtype=torch.float32), empty(1, dtype=torch.float32)
        s["dlogits"] = empty(rows, vocab)
        s["workspace"] = empty(1 << 20, dtype=torch.uint8)
    return s


def _workspace(case, backward):
    """Bytes of scratch enough for either direction: states of every 128 rows of every head, and the
    gradients of shared heads in 32 bits."""
    b, t, h, d = (case[n] for n in ("batch", "seq", "heads", "dim"))
    parts = -(-t // 128)
    one = 4 * b * h * parts * d * d
    return 3 * one + 2 * 4 * b * t * h * d if backward else one


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
CHUNK = 128


def _heads_first(x, heads, t_pad, lens):
    """[b, t, heads', d] as float32 [b, heads, t_pad, d], zero behind each sequence's length."""
    b, t, hx, d = x.shape
    x = x.float()
    if lens is not None:
        live = torch.arange(t, device=x.device)[None, :] < lens[:, None]
        x = torch.where(live[:, :, None, None], x, torch.zeros_like(x))
    x = x.transpose(1, 2)
    if hx != heads:
        x = x.repeat_interleave(heads // hx, dim=1)
    return torch.nn.functional.pad(x, (0, 0, 0, t_pad - t)).contiguous()


def _decayed_products(x, y, z, g, reverse=False):
    """out_i = sum over j <= i (reverse: j >= i) of exp(g |i - j|) (x_i . y_j) z_j, in chunks."""
    b, h, t, d = x.shape
    n = t // CHUNK
    x, y, z = (a.reshape(b, h, n, CHUNK, d) for a in (x, y, z))
    i = torch.arange(CHUNK, device=x.device, dtype=torch.float32)
    far = i[:, None] - i[None, :]
    far = -far if reverse else far
    decay = torch.where(far >= 0, torch.exp(g[:, None, None] * far.clamp(min=0)), torch.zeros((), device=x.device))
    to_end, from_start = (i + 1, CHUNK - 1 - i) if reverse else (CHUNK - 1 - i, i + 1)
    near = torch.matmul(torch.matmul(x, y.transpose(-1, -2).contiguous()) * decay[:, None], z)
    sums = torch.matmul((y * torch.exp(g[:, None, None, None] * to_end[:, None])).transpose(-1, -2).contiguous(), z)
    c = torch.arange(n, device=x.device, dtype=torch.float32)
    gap = c[:, None] - c[None, :] - 1
    gap = -gap - 2 if reverse else gap
    carry = torch.where(gap >= 0, torch.exp(g[:, None, None] * CHUNK * gap.clamp(min=0)), torch.zeros((), device=x.device))
    states = torch.matmul(carry, sums.reshape(b, h, n, d * d)).reshape(b, h, n, d, d)
    out = near + torch.matmul(x, states) * torch.exp(g[:, None, None, None] * from_start[:, None])
    return out.reshape(b, h, t, d)


def _ages(s, t_pad):
    """Rows' distances from the start, counted from 1, and from the end of their sequences, [b, t_pad]; the
    latter with False behind the ends."""
    b, t = s["batch"], s["seq"]
    lens = s["lens"] if s["lens"] is not None else torch.full((b,), t, device=DEV, dtype=torch.int32)
    at = torch.arange(t_pad, device=DEV, dtype=torch.float32)[None, :]
    left = lens[:, None].float() - 1 - at
    return at + 1, left.clamp(min=0), left >= 0, lens


def _last_state(y, z, g, left, live, weight, start, length):
    """sum_j weight_j y_j^T z_j + exp(g length) start."""
    w = torch.exp(g[None, :, None] * weight[:, None, :]) * live[:, None, :]
    state = torch.matmul((y * w[..., None]).transpose(-1, -2).contiguous(), z)
    return state + torch.exp(g[None, :] * length[:, None].float())[..., None, None] * start


def _merge(x, heads, t, dtype):
    """[b, h, t_pad, d] back to [b, t, heads, d], summed over the query heads that share one."""
    b, h, _, d = x.shape
    x = x[:, :, :t].reshape(b, heads, h // heads, t, d)
    return x.sum(2).transpose(1, 2).to(dtype).contiguous()


def _plain_fwd(s):
    t, h, g, dt = s["seq"], s["heads"], s["decay"], DTYPES[s["dtype"]]
    t_pad = -(-t // CHUNK) * CHUNK
    q, k, v = (_heads_first(s[n], h, t_pad, s["lens"]) for n in "qkv")
    o = _decayed_products(q, k, v, g)
    if s["state_in"] is None:
        return _merge(o * s["scale"], h, t, dt)
    age, left, live, lens = _ages(s, t_pad)
    o = o + torch.matmul(q, s["state_in"]) * torch.exp(g[None, :, None] * age[:, None])[..., None]
    return _merge(o * s["scale"], h, t, dt), _last_state(k, v, g, left, live, left, s["state_in"], lens)


def _plain_bwd(s):
    t, h, hk, g, dt, scale = s["seq"], s["heads"], s["kv"], s["decay"], DTYPES[s["dtype"]], s["scale"]
    t_pad = -(-t // CHUNK) * CHUNK
    q, k, v, do = (_heads_first(s[n], h, t_pad, s["lens"]) for n in ("q", "k", "v", "d_o"))
    dq = _decayed_products(do, v, k, g) * scale
    dk = _decayed_products(v, do, q, g, True) * scale
    dv = _decayed_products(k, q, do, g, True) * scale
    if s["state_in"] is None:
        return _merge(dq, h, t, dt), _merge(dk, hk, t, dt), _merge(dv, hk, t, dt)
    age, left, live, lens = _ages(s, t_pad)
    behind = torch.exp(g[None, :, None] * age[:, None])[..., None]
    ahead = (torch.exp(g[None, :, None] * left[:, None]) * live[:, None])[..., None]
    dq = dq + torch.matmul(do, s["state_in"].transpose(-1, -2).contiguous()) * behind * scale
    dk = dk + torch.matmul(v, s["d_state_out"].transpose(-1, -2).contiguous()) * ahead
    dv = dv + torch.matmul(k, s["d_state_out"]) * ahead
    first = _last_state(q * scale, do, g, left, live, age.expand_as(left), s["d_state_out"], lens)
    return _merge(dq, h, t, dt), _merge(dk, hk, t, dt), _merge(dv, hk, t, dt), first


def _plain_step(s):
    h, dt = s["heads"], DTYPES[s["dtype"]]
    q, k, v = (_heads_first(s[n], h, 1, None) for n in "qkv")
    state = torch.exp(s["decay"])[None, :, None, None] * s["state_in"] + k.transpose(-1, -2) * v
    return _merge((q.transpose(-1, -2) * state).sum(-2, keepdim=True) * s["scale"], h, 1, dt), state


def _gate_of_rows(s, rows):
    if s["gate"] is None:
        return torch.ones((), device=DEV)
    return s["gate"].float().repeat_interleave(s["gate_rows"], dim=0) if s["gate"].shape[0] > 1 else s["gate"].float()


def _plain_join(s):
    b, dt = s["b"].float(), DTYPES[s["dtype"]]
    gate = _gate_of_rows(s, b.shape[0])
    out = {}
    if s["post"]:
        out["rstd_post"] = torch.rsqrt(b.square().mean(1) + EPS)
        b = b * out["rstd_post"][:, None] * s["gamma_post"].float()
    h = s["alpha"] * s["x"].float() + gate * b
    out["rstd_pre"] = torch.rsqrt(h.square().mean(1) + EPS)
    out["h"], out["y"] = h.to(dt), (h * out["rstd_pre"][:, None] * s["gamma_pre"].float()).to(dt)
    return out


def _plain_join_bwd(s):
    dt = DTYPES[s["dtype"]]
    b, h, dy = s["b"].float(), s["h"].float(), s["dy"].float()
    gate = _gate_of_rows(s, b.shape[0])
    r = s["rstd_pre"][:, None]
    h = h * r
    t = dy * s["gamma_pre"].float()
    total = s["dh"].float() + r * (t - h * (t * h).mean(1, keepdim=True))
    out = {"dx": (s["alpha"] * total).to(dt), "dgamma_pre": (dy * h).sum(0)}
    gamma = s["gamma_post"].float() if s["post"] else torch.ones((), device=DEV)
    u = total * gate * gamma
    if s["post"]:
        r = s["rstd_post"][:, None]
        b = b * r
        out["db"] = (r * (u - b * (u * b).mean(1, keepdim=True))).to(dt)
        out["dgamma_post"] = (total * gate * b).sum(0)
    else:
        out["db"] = u.to(dt)
    if s["gate"] is not None:
        out["dgate"] = (total * gamma * b).reshape(s["gate"].shape[0], -1, b.shape[1]).sum(1)
    return out


def _plain_distill(s):
    z, tau = s["logits"].float() / s["temperature"], s["temperature"]
    ids, w = s["ids"].long(), s["weight"][:, None]
    z = z - z.max(1, keepdim=True).values
    e = torch.exp(z)
    total = e.sum(1, keepdim=True)
    teach = s["teacher"] / tau
    teach = teach - teach.max(1, keepdim=True).values
    p = torch.exp(teach)
    mass = p.sum(1, keepdim=True)
    p = p / mass
    log_ratio = teach - torch.log(mass) - (torch.gather(z, 1, ids) - torch.log(total))
    row = w[:, 0] * tau * tau * (p * log_ratio).sum(1)
    grad = (e / total).scatter_add(1, ids, -p) * (s["scale"] * tau * w)
    return {"row_loss": row, "loss": (row.sum() * s["scale"]).reshape(1), "dlogits": grad.to(DTYPES[s["dtype"]])}


PLAIN = {"linattn_fwd": _plain_fwd, "linattn_bwd": _plain_bwd, "linattn_step": _plain_step, "join_fwd": _plain_join,
         "join_bwd": _plain_join_bwd, "distill": _plain_distill}


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------
def _p(t):
    return None if t is None else t.data_ptr()


def _own(s):
    from jaxpp_amd import runtime as rt
    stream, f32, op = torch.cuda.current_stream().cuda_stream, s["dtype"] == "f32", s["op"]
    if op.startswith("linattn"):
        h, hk, d = s["heads"], s["kv"], s["dim"]
        sizes = dict(batch=s["batch"], n_heads=h, n_kv_heads=hk, head_dim=d, scale=s["scale"], f32=f32, stream=stream)
        if op == "linattn_step":
            rt.linattn_step(_p(s["q"]), _p(s["k"]), _p(s["v"]), _p(s["o"]), _p(s["decay"]), _p(s["state_in"]),
                            _p(s["state_out"]), h * d, hk * d, hk * d, h * d, **sizes)
            return s["o"], s["state_out"]
        sizes.update(seq=s["seq"], lens=_p(s["lens"]), workspace=_p(s["workspace"]), state_in=_p(s["state_in"]))
        if op == "linattn_fwd":
            rt.linattn_fwd(_p(s["q"]), _p(s["k"]), _p(s["v"]), _p(s["o"]), _p(s["decay"]), h * d, hk * d, hk * d, h * d,
                           state_out=_p(s["state"]), **sizes)
            return s["o"] if s["state"] is None else (s["o"], s["state"])
        rt.linattn_bwd(_p(s["q"]), _p(s["k"]), _p(s["v"]), _p(s["d_o"]), _p(s["dq"]), _p(s["dk"]), _p(s["dv"]),
                       _p(s["decay"]), h * d, hk * d, hk * d, h * d, h * d, hk * d, hk * d,
                       d_state_out=_p(s["d_state_out"]), d_state_in=_p(s["state"]), **sizes)
        grads = s["dq"], s["dk"], s["dv"]
        return grads if s["state"] is None else grads + (s["state"],)
    if op.startswith("join"):
        rows, cols = s["b"].shape
        common = dict(gamma_post=_p(s["gamma_post"]), gate=_p(s["gate"]), gate_rows=s["gate_rows"],
                      gamma_pre=_p(s["gamma_pre"]), rstd_post=_p(s["rstd_post"]) if s["post"] else None,
                      rstd_pre=_p(s["rstd_pre"]), alpha=s["alpha"], f32=f32, stream=stream)
        if op == "join_fwd":
            rt.block_join_fwd(_p(s["x"]), _p(s["b"]), _p(s["h"]), rows, cols, y=_p(s["y"]), eps=EPS, **common)
            return {n: s[n] for n in ("h", "y", "rstd_pre") + (("rstd_post",) if s["post"] else ())}
        rt.block_join_bwd(_p(s["h"]), _p(s["b"]), _p(s["dh"]), _p(s["dy"]), _p(s["dx"]), _p(s["db"]), rows, cols,
                          dgamma_post=_p(s["dgamma_post"]), dgate=_p(s["dgate"]), dgamma_pre=_p(s["dgamma_pre"]),
                          workspace=_p(s["workspace"]), accumulate=False, **common)
        return {n: s[n] for n in ("dx", "db", "dgamma_pre", "dgamma_post", "dgate") if s[n] is not None}
    rows, vocab = s["logits"].shape
    rt.distill_loss(_p(s["logits"]), _p(s["ids"]), _p(s["teacher"]), rows, vocab, s["ids"].shape[1], vocab,
                    _p(s["row_loss"]), loss=_p(s["loss"]), dlogits=_p(s["dlogits"]), ldd=vocab, weight=_p(s["weight"]),
                    temperature=s["temperature"], scale=s["scale"], workspace=_p(s["workspace"]), f32=f32, stream=stream)
    return {n: s[n] for n in ("row_loss", "loss", "dlogits")}


def run(state):
    return _own(state) if own else PLAIN[state["op"]](state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    if case["op"].startswith("linattn"):
        b, t, h, hk, d = (case[n] for n in ("batch", "seq", "heads", "kv", "dim"))
        wide, shared, state = b * t * h * d * es, b * t * hk * d * es, 4 * b * h * d * d
        products = 2 * b * t * h * d * d
        if case["op"] == "linattn_step":
            return {"bytes": 2 * wide + 2 * shared + 2 * state, "flops": 2 * products}
        states = 2 * state if case["states"] else 0
        if case["op"] == "linattn_fwd":
            return {"bytes": 2 * wide + 2 * shared + states, "flops": 2 * products}
        return {"bytes": 3 * wide + 4 * shared + 1.5 * states, "flops": 5 * products}
    if case["op"].startswith("join"):
        n = case["batch"] * case["seq"] * case["cols"]
        moved = 4 if case["op"] == "join_fwd" else 6
        return {"bytes": moved * n * es, "flops": (12 if case["op"] == "join_fwd" else 30) * n}
    n = case["rows"] * case["vocab"]
    return {"bytes": 2 * n * es + 8 * case["rows"] * case["k"], "flops": 6 * n}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"l": _exact_linattn, "j": _exact_join, "d": _exact_distill}[case["op"][0]](s)


def _exact_linattn(s):
    """Sequence by sequence and head by head, every pair of rows for itself."""
    b, t, h, hk, d, scale = s["batch"], s["seq"], s["heads"], s["kv"], s["dim"], s["scale"]
    backward, states = s["op"] == "linattn_bwd", s["state_in"] is not None
    zeros = lambda like: torch.zeros(like.shape, dtype=torch.float64, device=DEV)
    dq, dk, dv, o = zeros(s["q"]), zeros(s["k"]), zeros(s["v"]), zeros(s["q"])
    last = torch.zeros(b, h, d, d, dtype=torch.float64, device=DEV)
    lens = [t] * b if s["lens"] is None else s["lens"].tolist()
    for ib, n in enumerate(lens):
        at = torch.arange(n, device=DEV, dtype=torch.float64)
        for ih in range(h):
            g, ik = s["decay"][ih].double(), ih // (h // hk)
            q, k, v = s["q"][ib, :n, ih].double(), s["k"][ib, :n, ik].double(), s["v"][ib, :n, ik].double()
            start = s["state_in"][ib, ih].double() if states else None
            down = torch.exp(g * (at + 1))[:, None]
            up = torch.exp(g * (n - 1 - at))[:, None]
            rows = 4096
            if not backward:
                for r in range(0, n, rows):
                    e = min(n, r + rows)
                    w = (at[r:e, None] - at[None, :e]) * g
                    pairs = (q[r:e] @ k[:e].T) * torch.where(at[r:e, None] >= at[None, :e], torch.exp(w), 0.0)
                    o[ib, r:e, ih] = scale * (pairs @ v[:e])
                if states:
                    o[ib, :n, ih] += scale * down * (q @ start)
                    last[ib, ih] = torch.exp(g * n) * start + (k * up).T @ v
                continue
            do = s["d_o"][ib, :n, ih].double()
            for r in range(0, n, rows):
                e = min(n, r + rows)
                w = scale * torch.where(at[r:e, None] >= at[None, :e], torch.exp((at[r:e, None] - at[None, :e]) * g), 0.0)
                d_pairs = (do[r:e] @ v[:e].T) * w
                dq[ib, r:e, ih] = d_pairs @ k[:e]
                dk[ib, :e, ik] += d_pairs.T @ q[r:e]
                dv[ib, :e, ik] += ((q[r:e] @ k[:e].T) * w).T @ do[r:e]
            if states:
                end = s["d_state_out"][ib, ih].double()
                dq[ib, :n, ih] += scale * down * (do @ start.T)
                dk[ib, :n, ik] += up * (v @ end.T)
                dv[ib, :n, ik] += up * (k @ end)
                last[ib, ih] = torch.exp(g * n) * end + scale * (q * down).T @ do
    if backward:
        return (dq, dk, dv, last) if states else (dq, dk, dv)
    return (o, last) if states else o


def _exact_join(s):
    wide = {n: s[n].double() for n in ("x", "b", "h", "dh", "dy", "gamma_post", "gamma_pre", "gate", "rstd_post", "rstd_pre")
            if isinstance(s.get(n), torch.Tensor)}
    rows, cols = wide["b"].shape
    gate = torch.ones(rows, cols, dtype=torch.float64, device=DEV)
    if s["gate"] is not None:
        for i in range(s["gate"].shape[0]):
            gate[i * s["gate_rows"]:(i + 1) * s["gate_rows"]] = wide["gate"][i]
    if s["op"] == "join_fwd":
        norm, out = wide["b"], {}
        if s["post"]:
            out["rstd_post"] = 1 / torch.sqrt((norm * norm).sum(1) / cols + EPS)
            norm = torch.einsum("rc,r,c->rc", norm, out["rstd_post"], wide["gamma_post"])
        out["h"] = s["alpha"] * wide["x"] + gate * norm
        out["rstd_pre"] = 1 / torch.sqrt((out["h"] ** 2).sum(1) / cols + EPS)
        out["y"] = torch.einsum("rc,r,c->rc", out["h"], out["rstd_pre"], wide["gamma_pre"])
        return out

    def norm_back(cot, x, r, gamma):
        """d(x r(x) gamma) for the cotangent, with the row scales r as given."""
        scaled = cot * gamma
        inner = (scaled * x).sum(1) * r ** 3 / cols
        return scaled * r[:, None] - x * inner[:, None]

    total = wide["dh"] + norm_back(wide["dy"], wide["h"], wide["rstd_pre"], wide["gamma_pre"])
    out = {"dx": s["alpha"] * total, "dgamma_pre": (wide["dy"] * wide["h"] * wide["rstd_pre"][:, None]).sum(0)}
    into = total * gate
    norm = wide["b"]
    if s["post"]:
        out["db"] = norm_back(into, wide["b"], wide["rstd_post"], wide["gamma_post"])
        norm = wide["b"] * wide["rstd_post"][:, None]
        out["dgamma_post"] = (into * norm).sum(0)
        norm = norm * wide["gamma_post"]
    else:
        out["db"] = into
    if s["gate"] is not None:
        rows_of = range(0, rows, s["gate_rows"])
        out["dgate"] = torch.stack([(total * norm)[i:i + s["gate_rows"]].sum(0) for i in rows_of])
    return out


def _exact_distill(s):
    """A few rows at a time."""
    tau, rows = s["temperature"], s["logits"].shape[0]
    row_loss = torch.zeros(rows, dtype=torch.float64, device=DEV)
    grad = torch.empty(s["logits"].shape, dtype=torch.float64, device=DEV)
    for r in range(0, rows, 256):
        at = slice(r, min(rows, r + 256))
        log_q = torch.log_softmax(s["logits"][at].double() / tau, dim=1)
        log_p = torch.log_softmax(s["teacher"][at].double() / tau, dim=1)
        ids, w = s["ids"][at].long(), s["weight"][at].double()
        row_loss[at] = w * tau ** 2 * (log_p.exp() * (log_p - log_q.gather(1, ids))).sum(1)
        p = torch.zeros_like(log_q).scatter_(1, ids, log_p.exp())
        grad[at] = (log_q.exp() - p) * (w * s["scale"] * tau)[:, None]
    return {"row_loss": row_loss, "loss": row_loss.sum().reshape(1) * s["scale"], "dlogits": grad}
