"""Cases of the decayed linear attention and of the head norms with rotation.

Linear attention with a decay for each head, w = exp(log_decay), state S
``[d_k, d_v]`` of each (sequence, value head):

    S_t = w S_{t-1} + k_t v_t^T        o_t = scale S_t^T q_t

in its three calls (``recurrent``: one token a row, ``chunked``: prompts,
``backward``: the gradients), and the RMS norm of each query and key head with
the position rotation in the same pass, with its gradient.

``own`` False: ``run`` computes the plain form; True: the framework's calls.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_ES = {"f32": 4, "bf16": 2, "f16": 2}
_EPS = 1e-6


# ---- the cases --------------------------------------------------------------
def listed():
    return [
        # One user's next token: 32 states of 64 KiB; latency is what counts.
        _la("decode, one row", "recurrent", seqs=1, tokens=1, hq=16, hv=32),
        # A served batch's next token: 1 GB of states in and out.
        _la("decode, 256 rows", "recurrent", seqs=256, tokens=256, hq=16, hv=32),
        # Prompts of many lengths packed, each continuing from a state.
        _la("prompts, 64 packed", "chunked", seqs=64, tokens=131072, hq=16, hv=32, state=True),
        # One long document, as many key heads as value heads.
        _la("prompt, one long", "chunked", seqs=1, tokens=32768, hq=32, hv=32),
        # A few short prompts of odd lengths (an empty one, a single token).
        _la("prompts, short", "chunked", seqs=5, tokens=331, hq=4, hv=8, state=True, dk=64, dv=64),
        # Full precision, as an evaluation against a reference runs.
        _la("prompts, f32", "chunked", seqs=8, tokens=8192, hq=8, hv=16, state=True, dtype="f32"),
        # A training batch's gradients.
        _la("gradient, batch", "backward", seqs=4, tokens=16384, hq=16, hv=16, packed=False),
        # Packed odd documents with shared key heads, gradients in f32.
        _la("gradient, f32", "backward", seqs=7, tokens=1501, hq=4, hv=8, state=True, dtype="f32", dk=64, dv=64),
        # q and k of a prompt, cut out of one fused projection.
        _nr("norm + rotation, prompt", "rope", tokens=32768, hq=16, hk=16, d=128, rot=128),
        # One token of each of 16 requests; a quarter of each head rotated.
        _nr("norm + rotation, decode", "rope", tokens=16, hq=16, hk=4, d=256, rot=64, dtype="f16"),
        # Its gradients over a training batch.
        _nr("norm + rotation, gradient", "rope_backward", tokens=16384, hq=16, hk=16, d=128, rot=128),
        # Odd token count, interleaved pairs, f32.
        _nr("norm + rotation, gradient f32", "rope_backward", tokens=777, hq=8, hk=4, d=96, rot=48, dtype="f32",
            interleaved=True),
    ]


def _la(name, op, seqs, tokens, hq, hv, state=None, dk=128, dv=128, dtype="bf16", packed=True):
    state = op == "recurrent" if state is None else state
    return {"name": name, "op": op, "seqs": seqs, "tokens": tokens, "heads_qk": hq, "heads_v": hv, "dk": dk, "dv": dv,
            "state": state, "packed": packed, "dtype": dtype}


def _nr(name, op, tokens, hq, hk, d, rot, dtype="bf16", interleaved=False):
    return {"name": name, "op": op, "tokens": tokens, "heads_q": hq, "heads_k": hk, "d": d, "rot": rot, "dtype": dtype,
            "interleaved": interleaved}


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["recurrent", "chunked", "chunked", "backward", "rope", "rope_backward"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f16", "f32"])
    if op in ("rope", "rope_backward"):
        d = rng.choice([64, 80, 96, 128, 128, 256])
        c = _nr("", op, _log(rng, 1, 16384), rng.choice([4, 8, 16, 32]), rng.choice([1, 2, 4, 8, 16]), d,
                rng.choice([d // 4, d // 2, d]), dtype, rng.random() < 0.3)
    else:
        dk, dv = rng.choice([(128, 128), (128, 128), (128, 128), (64, 64), (64, 128), (96, 96), (40, 72)])
        hq = rng.choice([2, 4, 8, 16])
        hv = hq * rng.choice([1, 1, 2, 4])
        if op == "recurrent":
            seqs = _log(rng, 1, 128)
            c = _la("", op, seqs, seqs, hq, min(hv, 32), None, dk, dv, dtype)
        else:
            tokens = _log(rng, 1, (32768 if dtype == "bf16" else 8192) if op == "chunked" else 8192)
            seqs = _log(rng, 1, min(64, tokens))
            packed = rng.random() < 0.7
            c = _la("", op, seqs, tokens if packed else -(-tokens // seqs) * seqs, hq, hv, rng.random() < 0.5, dk, dv,
                    dtype, packed)
    del c["name"]
    return c


# ---- inputs -----------------------------------------------------------------
def _lengths(case):
    """Lengths of a pack: lognormal, summing to `tokens`; zeros and ones occur
    in packs of short sequences."""
    n, total = case["seqs"], case["tokens"]
    if case["op"] == "recurrent" or not case["packed"]:
        return [total // n] * n
    r = np.random.default_rng(n * 1000003 + total)
    x = r.lognormal(0.0, 1.0, n)
    x = np.floor(x * total / x.sum()).astype(np.int64)
    if n >= 4:
        x[1], x[2] = 0, 1
    i = int(np.argmax(x))
    x[i] += total - int(x.sum())
    return [int(v) for v in x]


def _make_la(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DT[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)

    t, n, hq, hv, dk, dv = (case[k] for k in ("tokens", "seqs", "heads_qk", "heads_v", "dk", "dv"))
    lens = _lengths(case)
    cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int64)
    # q and k as a head norm leaves them (root mean square 1); decays of a
    # geometric series over the heads, scaled by the layer, as slopes are set.
    rms = lambda x: x / x.square().mean(-1, keepdim=True).sqrt()  # noqa: E731
    layer = float(torch.rand(1, generator=g, device="cuda").item()) * 0.9 + 0.1
    slopes = torch.exp2(-8.0 * torch.arange(1, hv + 1, device="cuda", dtype=torch.float64) / hv)
    s = {"q": rms(normal(t, hq, dk)).to(dt), "k": rms(normal(t, hq, dk)).to(dt), "v": normal(t, hv, dv).to(dt),
         "log_decay": (-slopes * layer).float(), "scale": dk ** -0.5,
         "state": normal(n, hv, dk, dv) if case["state"] else None,
         "cu": torch.tensor(cu, dtype=torch.int32, device="cuda"), "lens": lens}
    if case["op"] == "backward":
        s["do"] = normal(t, hv, dv).to(dt)
        s["ds"] = normal(n, hv, dk, dv) * 0.1 if case["state"] else None
    if case["op"] == "recurrent":
        s["next"] = torch.empty_like(s["state"])  # the other of two state buffers
    return s, lens


def _chunk_rows(lens, size):
    """Token index of each (chunk, position), -1 past a sequence's end, and
    each chunk's sequence; chunks never span two sequences."""
    rows, seq, start = [], [], 0
    for i, n in enumerate(lens):
        k = -(-n // size)
        r = np.arange(k * size)
        rows.append(np.where(r < n, r + start, -1).reshape(k, size))
        seq += [i] * k
        start += n
    return np.concatenate(rows, 0), np.array(seq, dtype=np.int64)


def _make_nr(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DT[case["dtype"]]
    t, hq, hk, d, rot = (case[k] for k in ("tokens", "heads_q", "heads_k", "d", "rot"))

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)

    # q and k are parts of one projection's output [tokens, (hq + 2 hk) d].
    x = (normal(t, hq + 2 * hk, d) * 2.0).to(dt)
    table = 40960
    inv = 1e4 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
    ang = torch.arange(table, device="cuda", dtype=torch.float64)[:, None] * inv
    first = int(torch.randint(0, table - t, (1,), generator=g, device="cuda").item())
    s = {"q": x[:, :hq], "k": x[:, hq:hq + hk], "cos": ang.cos().float(), "sin": ang.sin().float(),
         "positions": torch.arange(first, first + t, device="cuda", dtype=torch.int32),
         "qw": 1.0 + 0.1 * normal(d), "kw": 1.0 + 0.1 * normal(d)}
    if case["op"] == "rope_backward":
        s["dq"], s["dk"] = normal(t, hq, d).to(dt), normal(t, hk, d).to(dt)
    return s


def prepare(case, seed):
    if case["op"] in ("rope", "rope_backward"):
        return {"case": case, **_make_nr(case, seed)}
    s, lens = _make_la(case, seed)
    if case["op"] != "recurrent":
        rows, seq = _chunk_rows(lens, 256 if case["tokens"] >= 8192 else 64)
        s["rows"] = torch.from_numpy(rows).cuda()
        s["seq"] = torch.from_numpy(seq).cuda()
        s["lens_dev"] = torch.tensor(lens, device="cuda")
    s.pop("lens")
    if case["op"] != "recurrent" and not case["packed"]:  # [B, T, H, d]
        n = case["seqs"]
        for key in ("q", "k", "v", "do"):
            if key in s:
                s[key] = s[key].reshape((n, -1) + s[key].shape[1:])
        s["cu"] = None
    return {"case": case, **s}


# ---- the plain forms ----------------------------------------------------------
def _gather(x, rows):
    """[T, H, d] -> [H, chunks, size, d] in f32, zeros past a sequence's end."""
    y = x.flatten(0, -3)[rows.clamp_min(0)].float()
    return (y * (rows >= 0)[..., None, None]).permute(2, 0, 1, 3)


def _scatter(y, rows, like):
    """The inverse: [H, chunks, size, d] -> like's shape and type."""
    out = torch.empty(like.shape, dtype=like.dtype, device=like.device)
    flat = out.view((-1,) + like.shape[-2:])
    keep = rows >= 0
    flat[rows[keep]] = y.permute(1, 2, 0, 3)[keep].to(like.dtype)
    return out


def _repeat(x, hv):
    return x.repeat_interleave(hv // x.shape[-2], dim=-2)


def _chunk_terms(s):
    """What both directions need: each chunk's valid count, and the powers of
    the decays inside a chunk and between chunks."""
    rows, seq = s["rows"], s["seq"]
    valid = (rows >= 0).sum(1)  # [chunks]
    g = s["log_decay"].double()
    size, n = rows.shape
    i = torch.arange(n, device=rows.device)
    dist = i[:, None] - i[None, :]
    intra = torch.where(dist >= 0, torch.exp(g[:, None, None] * dist.clamp_min(0)), 0.0).float()
    upto = rows.clamp_min(0).amax(1)  # last token of each chunk
    first = rows[:, 0]
    # Chunk b's contribution as it stands at the start of a later chunk a of
    # the same sequence: w^(first token of a - 1 - last token of b).
    gap = first[:, None] - 1 - upto[None, :]
    same = (seq[:, None] == seq[None, :]) & (gap >= 0)
    between = torch.where(same, torch.exp(g[:, None, None] * gap.clamp_min(0)), 0.0).float()
    return rows, seq, valid, g, i, intra, between, first, upto


def _starts(s, b):
    """[n_seqs] -> the number of tokens before each chunk in its sequence."""
    seq, first = s["seq"], s["rows"][:, 0]
    start = torch.cumsum(s["lens_dev"], 0) - s["lens_dev"]
    return (first - start[seq]).double()


def _plain_states(s, k, v, terms):
    """Each chunk's state before it [H, chunks, dk, dv], and the states after
    the sequences [n, H, dk, dv]."""
    rows, seq, valid, g, i, intra, between, first, upto = terms
    back = torch.exp(g[:, None, None] * (valid[:, None] - 1 - i).clamp_min(0)).float()  # w^(c-1-j)
    part = (k * back[..., None]).transpose(-1, -2) @ v  # [H, chunks, dk, dv]
    flat = part.flatten(2)
    before = (between @ flat).view_as(part)
    n, h = s["lens_dev"].numel(), g.numel()
    lens = s["lens_dev"].double()
    start = torch.cumsum(s["lens_dev"], 0) - s["lens_dev"]
    after = start[:, None] + s["lens_dev"][:, None] - 1 - upto[None, :]  # tokens from chunk b's end to the end
    mine = torch.arange(n, device=seq.device)[:, None] == seq[None, :]
    w = torch.where(mine, torch.exp(g[:, None, None] * after.clamp_min(0)), 0.0).float()
    final = (w @ flat).view(h, n, *part.shape[2:])
    if s["state"] is not None:
        s0 = s["state"].transpose(0, 1)
        before = before + torch.exp(g[:, None] * _starts(s, None)).float()[..., None, None] * s0[:, seq]
        final = final + torch.exp(g[:, None] * lens).float()[..., None, None] * s0
    return before, final.transpose(0, 1).contiguous()


def _plain_chunked(s):
    hv = s["log_decay"].numel()
    terms = _chunk_terms(s)
    rows, _, _, g, i, intra, *_ = terms
    q, k, v = (_gather(x, rows) for x in (_repeat(s["q"], hv), _repeat(s["k"], hv), s["v"]))
    before, final = _plain_states(s, k, v, terms)
    p = (q @ k.transpose(-1, -2)) * intra[:, None]
    o = p @ v + (q @ before) * torch.exp(g[:, None] * (i + 1)).float()[:, None, :, None]
    return _scatter(o * s["scale"], rows, s["v"]), final


def _plain_backward(s):
    hq, hv = s["q"].shape[-2], s["log_decay"].numel()
    terms = _chunk_terms(s)
    rows, seq, valid, g, i, intra, between, first, upto = terms
    q, k, v, do = (_gather(x, rows) for x in (_repeat(s["q"], hv), _repeat(s["k"], hv), s["v"], s["do"]))
    before, _ = _plain_states(s, k, v, terms)
    ahead = torch.exp(g[:, None] * (i + 1)).float()  # w^(i+1)
    # The state gradient as it reaches each chunk's end from later chunks.
    part = (q * (s["scale"] * ahead)[:, None, :, None]).transpose(-1, -2) @ do
    flat = part.flatten(2)
    later = (between.transpose(-1, -2) @ flat).view_as(part)
    n = s["lens_dev"].numel()
    start = torch.cumsum(s["lens_dev"], 0) - s["lens_dev"]
    mine = torch.arange(n, device=seq.device)[:, None] == seq[None, :]
    w0 = torch.where(mine, torch.exp(g[:, None, None] * (first[None, :] - start[:, None]).clamp_min(0)), 0.0).float()
    d_state = (w0 @ flat).view(hv, n, *part.shape[2:])
    if s["ds"] is not None:
        ds = s["ds"].transpose(0, 1)
        left = (start + s["lens_dev"])[seq] - 1 - upto
        later = later + torch.exp(g[:, None] * left).float()[..., None, None] * ds[:, seq]
        d_state = d_state + torch.exp(g[:, None] * s["lens_dev"]).float()[..., None, None] * ds
    back = torch.exp(g[:, None, None] * (valid[:, None] - 1 - i).clamp_min(0)).float()
    p = (q @ k.transpose(-1, -2)) * intra[:, None] * s["scale"]
    dp = (do @ v.transpose(-1, -2)) * intra[:, None] * s["scale"]
    dq = dp @ k + (do @ before.transpose(-1, -2)) * (s["scale"] * ahead)[:, None, :, None]
    dk = dp.transpose(-1, -2) @ q + (v @ later.transpose(-1, -2)) * back[..., None]
    dv = p.transpose(-1, -2) @ do + (k @ later) * back[..., None]
    share = lambda x: x.view(hq, hv // hq, *x.shape[1:]).sum(1)  # noqa: E731
    grads = [_scatter(share(dq), rows, s["q"]), _scatter(share(dk), rows, s["k"]), _scatter(dv, rows, s["v"])]
    return grads + ([d_state.transpose(0, 1).contiguous()] if s["state"] is not None else [])


def _plain_recurrent(s):
    hv = s["log_decay"].numel()
    q, k, v = _repeat(s["q"], hv).float(), _repeat(s["k"], hv).float(), s["v"].float()
    state = torch.exp(s["log_decay"])[:, None, None] * s["state"] + k[..., :, None] * v[..., None, :]
    o = (q[..., None, :] @ state)[..., 0, :] * s["scale"]
    return o.to(s["q"].dtype), state


def _rotate(x, cos, sin, rot, interleaved, sign=1.0):
    a, rest = x[..., :rot], x[..., rot:]
    if interleaved:
        x1, x2 = a[..., 0::2], a[..., 1::2]
        y = torch.stack([x1 * cos - sign * x2 * sin, x2 * cos + sign * x1 * sin], -1).flatten(-2)
    else:
        x1, x2 = a[..., : rot // 2], a[..., rot // 2:]
        y = torch.cat([x1 * cos - sign * x2 * sin, x2 * cos + sign * x1 * sin], -1)
    return torch.cat([y, rest], -1)


def _plain_rope(s):
    c = s["case"]
    cos, sin = (s[n][s["positions"].long()][:, None, :] for n in ("cos", "sin"))
    out = []
    for x, w in ((s["q"], s["qw"]), (s["k"], s["kw"])):
        y = x.float()
        y = y * (y.square().mean(-1, keepdim=True) + _EPS).rsqrt() * w
        out.append(_rotate(y, cos, sin, c["rot"], c["interleaved"]).to(x.dtype))
    return out


def _plain_rope_backward(s):
    c = s["case"]
    cos, sin = (s[n][s["positions"].long()][:, None, :] for n in ("cos", "sin"))
    dx, dw = [], []
    for x, w, dy in ((s["q"], s["qw"], s["dq"]), (s["k"], s["kw"], s["dk"])):
        y, dn = x.float(), _rotate(dy.float(), cos, sin, c["rot"], c["interleaved"], -1.0)
        r = (y.square().mean(-1, keepdim=True) + _EPS).rsqrt()
        dw.append((y * r * dn).sum((0, 1)))
        dn = dn * w
        dx.append((r * dn - y * r.pow(3) * (y * dn).mean(-1, keepdim=True)).to(x.dtype))
    return dx + dw


# ---- one pass -----------------------------------------------------------------
def run(state):
    s, op = state, state["case"]["op"]
    if not own:
        return {"recurrent": _plain_recurrent, "chunked": _plain_chunked, "backward": _plain_backward,
                "rope": _plain_rope, "rope_backward": _plain_rope_backward}[op](s)
    if op in ("rope", "rope_backward"):
        from bunsen_b200 import layer

        args = (s["q"], s["k"], s["positions"], s["cos"], s["sin"], s["qw"], s["kw"], _EPS)
        if op == "rope":
            return layer.qk_norm_rope(*args, interleaved=s["case"]["interleaved"])
        return layer.qk_norm_rope_backward(s["dq"], s["dk"], *args, interleaved=s["case"]["interleaved"])
    from bunsen_b200.linear_attention import LinearAttention

    rule = LinearAttention(scale=s["scale"])
    if op == "recurrent":  # one token a row: [rows, 1, H, d]
        out, nxt = rule.recurrent(s["q"][:, None], s["k"][:, None], s["v"][:, None], s["log_decay"], s["state"],
                                  state_out=s["next"])
        return out[:, 0], nxt
    if op == "chunked":
        return rule.chunked(s["q"], s["k"], s["v"], s["log_decay"], s["state"], cu_seqlens=s["cu"])
    dq, dk, dv, d_state = rule.backward(s["q"], s["k"], s["v"], s["log_decay"], s["do"], s["state"], s["ds"],
                                        cu_seqlens=s["cu"])
    return [dq, dk, dv] + ([d_state] if d_state is not None else [])


def work(case):
    es = _ES[case["dtype"]]
    if case["op"] in ("rope", "rope_backward"):
        n = case["tokens"] * (case["heads_q"] + case["heads_k"]) * case["d"]
        tables = case["tokens"] * (4 * case["rot"] + 4)
        passes = 2 if case["op"] == "rope" else 3
        return {"bytes": passes * n * es + tables, "flops": n * (8 if passes == 2 else 16)}
    t, hq, hv, dk, dv = (case[k] for k in ("tokens", "heads_qk", "heads_v", "dk", "dv"))
    states = case["seqs"] * hv * dk * dv * 4
    if case["op"] == "backward":
        io = t * (4 * hq * dk + 3 * hv * dv) * es
        return {"bytes": io + (3 * states if case["state"] else 0), "flops": 10 * t * hv * dk * dv}
    io = t * (2 * hq * dk + 2 * hv * dv) * es
    return {"bytes": io + states * (2 if case["state"] else 1), "flops": 4 * t * hv * dk * dv}


# ---- in 64 bits, from the definition --------------------------------------------
def _exact_la(case, seed):
    """Position by position, all sequences at once (longest first, so that the
    live ones are a prefix)."""
    s, lens = _make_la(case, seed)
    if max(lens) * (1 if case["op"] != "backward" else 2) > 40000:
        return None
    hq, hv, dk, dv, n = case["heads_qk"], case["heads_v"], case["dk"], case["dv"], case["seqs"]
    order = sorted(range(n), key=lambda i: -lens[i])
    start = torch.tensor([sum(lens[:i]) for i in order], device="cuda")
    long = np.array([lens[i] for i in order])
    rank = torch.tensor(np.argsort(order), device="cuda")
    w = torch.exp(s["log_decay"].double())[:, None, None]
    scale, back = s["scale"], case["op"] == "backward"

    def at(x, rows):
        y = x[rows].double()
        return y.repeat_interleave(hv // y.shape[1], 1) if y.shape[1] != hv else y

    def first(x):
        return x.double()[order] if x is not None else torch.zeros(n, hv, dk, dv, dtype=torch.float64, device="cuda")

    S = first(s["state"])
    out = torch.zeros(case["tokens"], hv, dk if back else dv, dtype=torch.float64, device="cuda")
    for t in range(int(long.max())):
        m = int((long > t).sum())
        rows = start[:m] + t
        S[:m].mul_(w).add_(at(s["k"], rows)[..., :, None] * at(s["v"], rows)[..., None, :])
        if back:
            out[rows] = (S[:m] @ at(s["do"], rows)[..., None])[..., 0] * scale
        else:
            out[rows] = (at(s["q"], rows)[..., None, :] @ S[:m])[..., 0, :] * scale
    lead = (n, -1) if case["op"] != "recurrent" and not case["packed"] else (-1,)
    if not back:
        return out.view(*lead, hv, dv), S[rank]
    D = first(s["ds"])
    dk_, dv_ = torch.zeros_like(out), torch.zeros(case["tokens"], hv, dv, dtype=torch.float64, device="cuda")
    for t in range(int(long.max()) - 1, -1, -1):
        m = int((long > t).sum())
        rows = start[:m] + t
        D[:m].add_(at(s["q"], rows)[..., :, None] * (at(s["do"], rows) * scale)[..., None, :])
        dk_[rows] = (D[:m] @ at(s["v"], rows)[..., None])[..., 0]
        dv_[rows] = (at(s["k"], rows)[..., None, :] @ D[:m])[..., 0, :]
        D[:m].mul_(w)
    share = lambda x: x.view(-1, hq, hv // hq, dk).sum(2).view(*lead, hq, dk)  # noqa: E731
    return [share(out), share(dk_), dv_.view(*lead, hv, dv)] + ([D[rank]] if case["state"] else [])


def _exact_nr(case, seed):
    """The rotation as complex numbers, the gradient through the definition."""
    s = _make_nr(case, seed)
    pos, half = s["positions"].long(), case["rot"] // 2
    turn = torch.complex(s["cos"][pos].double(), s["sin"][pos].double())[:, None, :]
    index = torch.arange(case["rot"], device="cuda").view(half, 2) if case["interleaved"] else \
        torch.arange(case["rot"], device="cuda").view(2, half).T

    def forward(x, u):
        y = x / torch.sqrt((x * x).sum(-1, keepdim=True) / case["d"] + _EPS) * u
        z = torch.complex(y[..., index[:, 0]], y[..., index[:, 1]]) * turn
        y = y.clone()
        y[..., index[:, 0]], y[..., index[:, 1]] = z.real, z.imag
        return y

    xs = [(s["q"].double(), s["qw"].double()), (s["k"].double(), s["kw"].double())]
    if case["op"] == "rope":
        return [forward(*a) for a in xs]
    dx, dw = [], []
    for (x, u), dy in zip(xs, (s["dq"], s["dk"])):
        x, u = x.detach().requires_grad_(), u.detach().requires_grad_()
        a, b = torch.autograd.grad(forward(x, u), (x, u), dy.double())
        dx.append(a)
        dw.append(b)
    return dx + dw


def exact(case, seed):
    return (_exact_nr if case["op"] in ("rope", "rope_backward") else _exact_la)(case, seed)
