"""Measured cases of self-attention's operators: norms of queries and keys with the
position rotation, causal attention with a window and sinks, and the paged cache of
serving (append, attention of a chunk of new tokens).

``own`` False computes every operator in its plain form (elementary torch
operations in 32 bits, angles in 64, rounded once at the end); ``own`` True makes the
calls a user's program makes of the package.  ``listed()`` holds the fixed cases and
``draw(rng)`` gives more of the same ranges.

Kinds:
  rotary_infer  qk_norm_rotary without autograd
  rotary_train  the same, forward and the gradients of q, k and the norms' weights
  window_infer  window_attention without autograd
  window_train  the same, forward and the gradients of q, k and v
  append        append_kv of new tokens to a paged cache, with their queries
  paged         paged_attention of new tokens over the pages
"""

from __future__ import annotations

import math
import random

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_EPS = 1e-6


# ------------------------------------------------------------------ cases

def _rotary(kind, B, N, H, Hk, D, rd, dtype="bf16", params="fp32", layout="seq", norm=True,
            interleaved=False, first=0, factor=1.0):
    """rd: rotated channels; first: the first token's position; factor: how far the
    frequencies are stretched for long contexts."""
    return {"kind": kind, "B": B, "N": N, "H": H, "Hk": Hk, "D": D, "rd": rd, "dtype": dtype,
            "params": params, "layout": layout, "norm": norm, "interleaved": interleaved,
            "first": first, "factor": factor}


def _window(kind, B, H, Hk, N, D, window=0, sinks=0, dtype="bf16", layout="seq", mask=False,
            empty=False):
    """window 0: all earlier tokens."""
    return {"kind": kind, "B": B, "H": H, "Hk": Hk, "N": N, "D": D, "window": window,
            "sinks": sinks, "dtype": dtype, "layout": layout, "mask": mask, "empty": empty}


def _append(S, new, ctx, H, Hk, D, rd, page, dtype="bf16", norm=True, interleaved=False):
    """S sequences of up to ``ctx`` states get up to ``new`` tokens each."""
    return {"kind": "append", "S": S, "new": new, "ctx": ctx, "H": H, "Hk": Hk, "D": D, "rd": rd,
            "page": page, "dtype": dtype, "norm": norm, "interleaved": interleaved}


def _paged(S, new, ctx, H, Hk, D, page, window=0, sinks=0, dtype="bf16", behind=0):
    """behind: rows of the batch that belong to no sequence."""
    return {"kind": "paged", "S": S, "new": new, "ctx": ctx, "H": H, "Hk": Hk, "D": D,
            "page": page, "window": window, "sinks": sinks, "dtype": dtype, "behind": behind}


def listed():
    return [
        # Queries and keys of a short prompt: launches and host time.
        {"name": "rotary_prompt", **_rotary("rotary_infer", 1, 77, 8, 8, 64, 64, "fp16")},
        # A training step's queries and keys, four query heads to a kv head.
        {"name": "rotary_train", **_rotary("rotary_train", 2, 4096, 32, 8, 128, 128)},
        # FP32, neighbouring channels as pairs, half of an odd head size rotated, positions
        # far into a stretched context.
        {"name": "rotary_odd", **_rotary("rotary_train", 3, 1021, 6, 2, 72, 36, "fp32", "fp32",
                                         "head", True, True, 1000003, 8.0)},
        # A short prompt, all earlier tokens visible: launches and host time.
        {"name": "window_prompt", **_window("window_infer", 1, 8, 8, 77, 64, dtype="fp16")},
        # A training batch as it comes: odd lengths, padding, a sequence with no tokens at all.
        {"name": "window_ragged",
         **_window("window_train", 4, 16, 4, 1021, 80, 300, 7, mask=True, empty=True)},
        # The training of a long context with a window and four tokens that stay visible.
        {"name": "window_long", **_window("window_train", 1, 16, 4, 16384, 64, 1024, 4)},
        # The largest training call: all earlier tokens, four query heads to a kv head.
        {"name": "window_train", **_window("window_train", 2, 32, 8, 4096, 128, layout="head")},
        # The new tokens of a decoding batch, one each.
        {"name": "append_token", **_append(16, 1, 8190, 32, 8, 128, 128, 64)},
        # Chunks of prompts, small pages, a part of each head rotated, FP16.
        {"name": "append_chunk", **_append(8, 1024, 4096, 16, 16, 80, 40, 16, "fp16", False, True)},
        # One decoded token of one short sequence: launches and host time.
        {"name": "token_short", **_paged(1, 1, 76, 8, 8, 64, 16)},
        # One token for each of 16 sequences of ragged long contexts: the states' bytes.
        {"name": "token_long", **_paged(16, 1, 8190, 32, 8, 128, 64)},
        # Chunks of prompts between decoded tokens, window and sinks, FP16, odd pages, rows
        # behind the last sequence.
        {"name": "chunk_window", **_paged(8, 512, 6000, 16, 4, 96, 48, 2048, 16, "fp16", 100)},
    ]


def _log_size(rng, lo, hi):
    """A size from lo to hi, even over its logarithm; a quarter of them
    multiples of 64."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if n >= 64 and rng.random() < 0.25:
        n = (n + 32) // 64 * 64
    return max(lo, min(hi, n))


def draw(rng):
    kind = rng.choice(["rotary_infer", "rotary_train", "rotary_train", "window_infer",
                       "window_train", "window_train", "append", "append", "paged", "paged",
                       "paged"])
    G = rng.choice([1, 1, 2, 3, 4, 8])
    Hk = rng.choice([1, 2, 4, 8])
    D = rng.choice([32, 40, 64, 64, 80, 96, 128, 128])
    rd = rng.choice([D, D, D // 2, D // 4 * 2])
    inter = rng.random() < 0.3
    if kind.startswith("rotary"):
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        width = (G + 1) * Hk * D
        most = 1 << 24 if dtype == "fp32" else 1 << 25
        N = _log_size(rng, 1, min(16384, most // width))
        B = rng.choice([1, 1, 2, 3, 8])
        while B > 1 and B * N * width > most:
            B -= 1
        return _rotary(kind, B, N, G * Hk, Hk, D, rd, dtype, rng.choice([dtype, "fp32"]),
                       rng.choice(["seq", "head"]), rng.random() < 0.7, inter,
                       rng.choice([0, 0, _log_size(rng, 100, 4000000)]),
                       rng.choice([1.0, 4.0, 16.0]))
    if kind.startswith("window"):
        train = kind == "window_train"
        N = _log_size(rng, 1, 16384)
        window = rng.choice([0, _log_size(rng, 1, 4096)])
        sinks = rng.choice([0, 0, 1, 4, 64, 200])
        B = rng.choice([1, 2, 4, 8])
        while True:
            case = _window(kind, B, G * Hk, Hk, N, D, window, sinks,
                           "bf16" if train else rng.choice(["bf16", "fp16"]),
                           rng.choice(["head", "seq"]), rng.random() < 0.5,
                           B > 1 and rng.random() < 0.25)
            if B * G * Hk * _pairs(N, window, sinks) <= 1 << 28 and B * G * Hk * N * D <= 1 << 25:
                return case
            if B > 1:
                B //= 2
            else:
                N = N * 2 // 3 + 1
    page = rng.choice([8, 16, 16, 32, 48, 64, 100, 256])
    new = rng.choice([1, 1, _log_size(rng, 2, 1024)])
    ctx = _log_size(rng, 1, 32768)
    S = _log_size(rng, 1, 64)
    dtype = rng.choice(["bf16", "fp16"])
    while S > 1 and (S * (ctx + new) * Hk * D > 1 << 27 or S * new * (G + 2) * Hk * D > 1 << 25
                     or S * new * G * Hk * (ctx + new) > 1 << 28):
        S //= 2
    if kind == "append":
        return _append(S, new, ctx, G * Hk, Hk, D, rd, page, dtype, rng.random() < 0.6, inter)
    while new * G * Hk * (ctx + new) > 1 << 28:
        new //= 2
    return _paged(S, new, ctx, G * Hk, Hk, D, page, rng.choice([0, 0, _log_size(rng, 1, 4096)]),
                  rng.choice([0, 4, 100]), dtype, rng.choice([0, 0, 1, 37]))


def _lengths(case):
    """(new tokens, states with them) of every sequence: ragged, the first one the
    longest; the same for every seed, so that the work is the case's own."""
    rng = random.Random(case["S"] * 1000003 + case["new"] * 1009 + case["ctx"])
    out = []
    for s in range(case["S"]):
        new = case["new"] if s == 0 or case["new"] == 1 else rng.randint(1, case["new"])
        ctx = case["ctx"] if s == 0 else rng.randint(case["ctx"] // 4, case["ctx"])
        out.append((new, ctx + new))
    return out


def _live(case):
    """Live tokens of every sequence of a padded batch."""
    rng = random.Random(case["B"] * 1009 + case["N"])
    live = [case["N"] - (rng.randint(0, case["N"] // 2) if case["mask"] else 0)
            for _ in range(case["B"])]
    if case["empty"] and case["mask"]:
        live[case["B"] // 2] = 0
    return live


def _seen(p, window, sinks, live=None):
    """States that the token at position p sees, of ``live`` ones (all up to p)."""
    top = p + 1 if live is None else min(p + 1, live)
    low = max(p + 1 - window, 0) if window else 0
    return max(top - low, 0) + max(min(low, sinks, top), 0)


def _pairs(N, window, sinks, live=None):
    return sum(_seen(p, window, sinks, live) for p in range(N))


# ----------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def _heads(g, case, h, n, dtype, scale=1.0):
    """[B, h, n, D], as a view of a [B, n, h, D] projection or head-major."""
    B, D = case["B"], case["D"]
    if case["layout"] == "seq":
        return (scale * _randn(g, B, n, h, D)).to(dtype).transpose(1, 2)
    return (scale * _randn(g, B, h, n, D)).to(dtype)


def _frequencies(rd, factor):
    """base^(-2c / rd), the slow ones divided by ``factor``: those that make at most one
    turn in 4096 tokens in full, those of 32 turns or more not at all, between them the
    division fades in with the turns."""
    f = torch.tensor([10000.0 ** (-2.0 * c / rd) for c in range(rd // 2)], dtype=torch.float64)
    if factor == 1.0:
        return f
    keep = ((4096 * f / (2.0 * math.pi) - 1.0) / 31.0).clamp(0.0, 1.0)
    return f * keep + f / factor * (1.0 - keep)


def _prepare_paged(case, g):
    """Sequences of ragged lengths over pages in random order; what no sequence has
    written holds earlier values."""
    D, Hk, page, dtype = case["D"], case["Hk"], case["page"], _TYPES[case["dtype"]]
    counts = _lengths(case)
    news, lengths = [n for n, _ in counts], [n for _, n in counts]
    starts = [sum(news[:s]) for s in range(len(news) + 1)]
    need = [-(-n // page) for n in lengths]
    pages = sum(need) + 3
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    tables = torch.zeros(len(need), max(need), dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(need):
        tables[s, :n] = order[at:at + n]
        at += n
    T = starts[-1] + case.get("behind", 0)
    state = {"k_cache": _randn(g, pages, Hk, page, D, dtype=dtype),
             "v_cache": _randn(g, pages, Hk, page, D, dtype=dtype), "tables": tables,
             "starts": torch.tensor(starts, dtype=torch.int32, device="cuda"),
             "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda"),
             "news": news, "counts": lengths, "first": starts,
             "q": (1.5 * _randn(g, T, case["H"], D)).to(dtype)}
    if case["kind"] == "append":
        state["k"], state["v"] = (_randn(g, T, Hk, D, dtype=dtype) for _ in range(2))
    if own:
        import openfold3_triangle_kernel_amd as tpf

        state["cache"] = tpf.PagedCache.of(state["k_cache"], state["v_cache"])
    return state


def prepare(case, seed):
    g = _gen(seed)
    kind, dtype = case["kind"], _TYPES[case["dtype"]]
    if kind.startswith("rotary"):
        B, N, H, Hk, D = (case[n] for n in ("B", "N", "H", "Hk", "D"))
        params = _TYPES[case["params"]]
        state = {"q": _heads(g, case, H, N, dtype, 1.5), "k": _heads(g, case, Hk, N, dtype),
                 "positions": torch.arange(case["first"], case["first"] + N, device="cuda").expand(B, N),
                 "frequencies": _frequencies(case["rd"], case["factor"]).cuda(),
                 "qw": None, "kw": None}
        if case["norm"]:
            state["qw"], state["kw"] = ((1.0 + 0.2 * _randn(g, D)).to(params) for _ in range(2))
        if kind == "rotary_train":
            state["dq"], state["dk"] = (_heads(g, case, h, N, dtype) for h in (H, Hk))
    elif kind.startswith("window"):
        B, N, H, Hk, D = (case[n] for n in ("B", "N", "H", "Hk", "D"))
        state = {"q": _heads(g, case, H, N, dtype, 1.5), "k": _heads(g, case, Hk, N, dtype),
                 "v": _heads(g, case, Hk, N, dtype), "mask": None}
        if case["mask"]:
            live = torch.tensor(_live(case), device="cuda")
            state["mask"] = torch.arange(N, device="cuda") < live[:, None]
        if kind == "window_train":
            state["dout"] = _randn(g, B, N, H, D, dtype=dtype)
    else:
        state = _prepare_paged(case, g)
        if kind == "append":
            D = case["D"]
            state["frequencies"] = _frequencies(case["rd"], 1.0).cuda()
            state["qw"], state["kw"] = (1.0 + 0.2 * _randn(g, D) for _ in range(2)) if case[
                "norm"] else (None, None)
    state["case"] = case
    return state


# ------------------------------------------------------------- plain forms

def _turn(x, cos, sin, interleaved, back=False):
    """The rotation of x [..., n, D] by cos and sin [..., n, rd / 2] (its transpose:
    ``back``)."""
    half = cos.shape[-1]
    if back:
        sin = -sin
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, x[..., 2 * half:]), -1)


def _plain_norm(x, w):
    rstd = 1.0 / torch.sqrt(x.square().mean(-1, keepdim=True) + _EPS)
    return x * rstd * w.float(), rstd


def _angles(positions, frequencies):
    angle = positions.double()[..., None] * frequencies
    return torch.cos(angle).float(), torch.sin(angle).float()


def _plain_rotary(state):
    case = state["case"]
    inter, norm = case["interleaved"], case["norm"]
    cos, sin = (t[:, None] for t in _angles(state["positions"], state["frequencies"]))
    out, grads = [], []
    for x_, w, dy in ((state["q"], state["qw"], state.get("dq")),
                      (state["k"], state["kw"], state.get("dk"))):
        x = x_.float()
        z, rstd = _plain_norm(x, w) if norm else (x, None)
        out.append(_turn(z, cos, sin, inter).to(x_.dtype))
        if dy is None:
            continue
        dz = _turn(dy.float(), cos, sin, inter, back=True)
        if norm:
            xh = x * rstd
            dw = (dz * xh).sum((0, 1, 2)).to(w.dtype)
            dz = dz * w.float()
            dz = rstd * (dz - xh * (dz * xh).mean(-1, keepdim=True))
            grads += [dz.to(x_.dtype), dw]
        else:
            grads.append(dz.to(x_.dtype))
    return out + grads


def _blocks(N, window, sinks, rows=512):
    """(first row, end, sinks before the rows' first state, first state) of blocks of
    rows: what a block's rows see lies in the states [0, head) and [low, end)."""
    for i in range(0, N, rows):
        end = min(N, i + rows)
        low = max(i + 1 - window, 0) if window else 0
        yield i, end, min(low, sinks), low


def _softmax(s):
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(top), 0.0, top))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total == 0, 1.0, total)  # a row without a state: zeros


def _plain_window(state):
    """Blocks of 512 rows against the states they may see; the query heads of a kv head
    are rows of one product."""
    case = state["case"]
    B, H, Hk, N, D = (case[n] for n in ("B", "H", "Hk", "N", "D"))
    G, window, sinks, dtype = H // Hk, case["window"], case["sinks"], state["q"].dtype
    scale = 1.0 / math.sqrt(D)
    q = state["q"].float().reshape(B, Hk, G, N, D)
    k, v = state["k"].float(), state["v"].float()
    train = case["kind"] == "window_train"
    out = torch.empty(B, Hk, G, N, D, device="cuda")
    if train:
        dout = state["dout"].float().transpose(1, 2).reshape(B, Hk, G, N, D)
        dq, dk, dv = torch.empty_like(out), torch.zeros_like(k), torch.zeros_like(v)
    for i, end, head, low in _blocks(N, window, sinks):
        pick = lambda t: torch.cat((t[:, :, :head], t[:, :, low:end]), 2)
        kb, vb = pick(k), pick(v)
        col = torch.cat((torch.arange(head, device="cuda"), torch.arange(low, end, device="cuda")))
        row = torch.arange(i, end, device="cuda")[:, None]
        see = col <= row
        if window:
            see = see & ((row - col < window) | (col < sinks))
        see = see.expand(B, end - i, len(col))
        if state["mask"] is not None:
            see = see & state["mask"][:, col][:, None]
        qb = q[:, :, :, i:end].reshape(B, Hk, G * (end - i), D)
        s = torch.matmul(qb, kb.transpose(-1, -2).contiguous()) * scale
        s = s.view(B, Hk, G, end - i, -1).masked_fill(~see[:, None, None], float("-inf"))
        p = _softmax(s).view(B, Hk, G * (end - i), -1)
        out[:, :, :, i:end] = torch.matmul(p, vb).view(B, Hk, G, end - i, D)
        if not train:
            continue
        do = dout[:, :, :, i:end].reshape(B, Hk, G * (end - i), D)
        dvb = torch.matmul(p.transpose(-1, -2).contiguous(), do)
        dp = torch.matmul(do, vb.transpose(-1, -2).contiguous())
        ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
        dq[:, :, :, i:end] = torch.matmul(ds, kb).view(B, Hk, G, end - i, D)
        dkb = torch.matmul(ds.transpose(-1, -2).contiguous(), qb)
        for total, part in ((dk, dkb), (dv, dvb)):
            total[:, :, :head] += part[:, :, :head]
            total[:, :, low:end] += part[:, :, head:]
    o = out.view(B, H, N, D).transpose(1, 2).to(dtype).contiguous()
    if not train:
        return [o]
    return [o, dq.view(B, H, N, D).to(dtype), dk.to(dtype), dv.to(dtype)]


def _plain_append(state):
    case = state["case"]
    page = case["page"]
    q, k, v = state["q"].float(), state["k"].float(), state["v"]
    where = torch.cat([torch.arange(n - new, n, device="cuda")
                       for new, n in zip(state["news"], state["counts"])])
    cos, sin = (t[:, None] for t in _angles(where, state["frequencies"]))
    if case["norm"]:
        q, k = _plain_norm(q, state["qw"])[0], _plain_norm(k, state["kw"])[0]
    q, k = (_turn(t, cos, sin, case["interleaved"]) for t in (q, k))
    at = 0
    for s, (new, n) in enumerate(zip(state["news"], state["counts"])):
        slot = torch.arange(n - new, n, device="cuda")
        pages = state["tables"][s].long()[slot // page]
        state["k_cache"][pages, :, slot % page] = k[at:at + new].to(v.dtype)
        state["v_cache"][pages, :, slot % page] = v[at:at + new]
        at += new
    return [q.to(v.dtype), state["k_cache"], state["v_cache"]]


def _plain_paged(state):
    case = state["case"]
    H, Hk, D, page, window, sinks = (case[n] for n in ("H", "Hk", "D", "page", "window", "sinks"))
    G, scale = H // Hk, 1.0 / math.sqrt(D)
    q = state["q"]
    out = torch.zeros_like(q)
    at = 0
    for s, (new, n) in enumerate(zip(state["news"], state["counts"])):
        pages = state["tables"][s, :-(-n // page)].long()
        k, v = (state[name][pages].transpose(0, 1).reshape(Hk, -1, D)[:, :n].float()
                for name in ("k_cache", "v_cache"))
        rows = q[at:at + new].float().view(new, Hk, G, D).permute(1, 2, 0, 3).reshape(Hk, G * new, D)
        scores = torch.matmul(rows, k.transpose(-1, -2).contiguous()) * scale
        col = torch.arange(n, device="cuda")
        row = torch.arange(n - new, n, device="cuda")[:, None]
        see = col <= row
        if window:
            see = see & ((row - col < window) | (col < sinks))
        scores = scores.view(Hk, G, new, n).masked_fill(~see, float("-inf"))
        o = torch.matmul(_softmax(scores).view(Hk, G * new, n), v)
        out[at:at + new] = o.view(Hk, G, new, D).permute(2, 0, 1, 3).reshape(new, H, D).to(q.dtype)
        at += new
    return [out]


def _plain(state):
    kind = state["case"]["kind"]
    if kind.startswith("rotary"):
        return _plain_rotary(state)
    if kind.startswith("window"):
        return _plain_window(state)
    return _plain_append(state) if kind == "append" else _plain_paged(state)


# ------------------------------------------------------ the package's calls

def _own(state):
    import openfold3_triangle_kernel_amd as tpf

    case = state["case"]
    kind = case["kind"]
    if kind == "append":
        q = tpf.append_kv(state["cache"], state["k"], state["v"], state["tables"], state["starts"],
                          state["lengths"], q=state["q"], frequencies=state["frequencies"],
                          q_weight=state["qw"], k_weight=state["kw"],
                          eps=_EPS if case["norm"] else None, interleaved=case["interleaved"])
        return [q, state["cache"].k, state["cache"].v]
    if kind == "paged":
        return [tpf.paged_attention(state["q"], state["cache"], state["tables"], state["starts"],
                                    state["lengths"], window=case["window"] or None,
                                    sinks=case["sinks"])]
    if kind.startswith("rotary"):
        names = ["q", "k"] + (["qw", "kw"] if case["norm"] else [])
        leaves = {n: state[n] for n in ("q", "k", "qw", "kw")}
        if kind == "rotary_train":
            leaves.update({n: state[n].detach().requires_grad_(True) for n in names})
        out = tpf.qk_norm_rotary(leaves["q"], leaves["k"], state["positions"], state["frequencies"],
                                 leaves["qw"], leaves["kw"], eps=_EPS if case["norm"] else None,
                                 interleaved=case["interleaved"])
        if kind == "rotary_infer":
            return list(out)
        order = ["q", "qw", "k", "kw"] if case["norm"] else ["q", "k"]
        grads = torch.autograd.grad(out, [leaves[n] for n in order], (state["dq"], state["dk"]))
        return [out[0].detach(), out[1].detach(), *grads]
    limits = {"window": case["window"] or None, "sinks": case["sinks"], "key_mask": state["mask"]}
    if kind == "window_infer":
        return [tpf.window_attention(state["q"], state["k"], state["v"], **limits)]
    leaves = [state[n].detach().requires_grad_(True) for n in "qkv"]
    out = tpf.window_attention(*leaves, **limits)
    return [out.detach(), *torch.autograd.grad(out, leaves, state["dout"])]


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------- work

def work(case):
    """Bytes: every input read and every output written once (of a cache the live states
    that the tokens see); operations of the products, or of the norm and rotation."""
    kind = case["kind"]
    size = torch.finfo(_TYPES[case["dtype"]]).bits // 8
    D, H, Hk = case["D"], case["H"], case["Hk"]
    if kind.startswith("rotary"):
        n = case["B"] * case["N"] * (H + Hk) * D
        if kind == "rotary_infer":
            return {"bytes": 2 * n * size, "flops": 8 * n}
        return {"bytes": 5 * n * size, "flops": 24 * n}
    if kind.startswith("window"):
        n = case["B"] * case["N"] * D * size
        pairs = H * sum(_pairs(case["N"], case["window"], case["sinks"], live) for live in _live(case))
        if kind == "window_infer":
            return {"bytes": n * (2 * H + 2 * Hk), "flops": 4 * pairs * D}
        return {"bytes": n * (4 * H + 4 * Hk), "flops": 14 * pairs * D}
    counts = _lengths(case)
    T = sum(new for new, _ in counts)
    if kind == "append":
        n = T * (2 * H + 4 * Hk) * D
        return {"bytes": n * size, "flops": 8 * T * (H + Hk) * D}
    window, sinks = case["window"], case["sinks"]
    states = sum(n - max(0, n - new + 1 - window - sinks) if window else n for new, n in counts)
    pairs = H * sum(_seen(p, window, sinks) for new, n in counts for p in range(n - new, n))
    return {"bytes": (2 * T * H + 2 * states * Hk) * D * size, "flops": 4 * pairs * D}


# ---------------------------------------------------------- 64-bit results

def _exact_turn(x, positions, frequencies, interleaved, back=False):
    """The pairs as complex numbers times exp(i angle); x [..., n, D], positions [n]."""
    half = len(frequencies)
    first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (
        slice(0, half), slice(half, 2 * half))
    angle = positions.to(torch.float64)[:, None] * frequencies
    spin = torch.polar(torch.ones_like(angle), -angle if back else angle)
    y = x.clone()
    z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * spin
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_rotary(case, s):
    out, grads = [], []
    positions = s["positions"][0]
    for name, w in (("q", s["qw"]), ("k", s["kw"])):
        x = s[name].double()
        r = torch.ones_like(x[..., :1]) if w is None else (
            torch.einsum("...d,...d->...", x, x)[..., None] / case["D"] + _EPS).rsqrt()
        scale = 1.0 if w is None else w.double()
        out.append(_exact_turn(x * r * scale, positions, s["frequencies"], case["interleaved"]))
        if case["kind"] != "rotary_train":
            continue
        dz = _exact_turn(s["d" + name].double(), positions, s["frequencies"], case["interleaved"], True)
        g = dz * scale
        if w is None:
            grads.append(g)
        else:
            dot = torch.einsum("...d,...d->...", g, x)[..., None]
            grads += [g * r - x * r.pow(3) * dot / case["D"], torch.einsum("bhnd,bhnd->d", dz, x * r)]
    return out + grads


def _exact_rows(q, k, v, positions, window, sinks, live, scale):
    """(probabilities, outputs) of one head's rows at ``positions`` over the states
    0 .. len(k) - 1 of which ``live`` count; rows that see none are 0."""
    col = torch.arange(k.shape[0], device="cuda")
    dead = col[None, :] > positions[:, None]
    if window:
        dead |= (positions[:, None] - col[None, :] >= window) & (col >= sinks)[None, :]
    dead |= ~live[None, :]
    logits = (q @ k.T) * scale
    logits[dead] = -torch.inf
    p = torch.softmax(logits, -1)
    p[dead.all(-1)] = 0.0
    return p, p @ v


def _exact_window(case, s):
    B, H, Hk, N, D = (case[n] for n in ("B", "H", "Hk", "N", "D"))
    train = case["kind"] == "window_train"
    scale = D ** -0.5
    at = torch.arange(N, device="cuda")
    out = torch.empty(B, N, H, D, dtype=torch.float64, device="cuda")
    dq = torch.empty(B, H, N, D, dtype=torch.float64, device="cuda")
    dk, dv = (torch.zeros(B, Hk, N, D, dtype=torch.float64, device="cuda") for _ in range(2))
    for b in range(B):
        live = torch.ones(N, dtype=torch.bool, device="cuda") if s["mask"] is None else s["mask"][b]
        for h in range(H):
            hk = h // (H // Hk)
            q, k, v = s["q"][b, h].double(), s["k"][b, hk].double(), s["v"][b, hk].double()
            p, out[b, :, h] = _exact_rows(q, k, v, at, case["window"], case["sinks"], live, scale)
            if not train:
                continue
            do = s["dout"][b, :, h].double()
            ds = do @ v.T
            ds -= torch.einsum("nd,nd->n", do, out[b, :, h])[:, None]
            ds *= p
            dq[b, h] = (ds @ k) * scale
            dk[b, hk] += (ds.T @ q) * scale
            dv[b, hk] += p.T @ do
    return [out, dq, dk, dv] if train else [out]


def _exact_places(case, s):
    """(sequence, token, position, page, place in it) of every new token."""
    tables, token = s["tables"].tolist(), 0
    for b, (new, n) in enumerate(_lengths(case)):
        for p in range(n - new, n):
            yield b, token, p, tables[b][p // case["page"]], p % case["page"]
            token += 1


def _exact_append(case, s):
    places = list(_exact_places(case, s))
    index = lambda i: torch.tensor([place[i] for place in places], device="cuda")
    token, positions, page, slot = (index(i) for i in (1, 2, 3, 4))
    turned = []
    for x, w in ((s["q"], s["qw"]), (s["k"], s["kw"])):
        x = x.double()
        if w is not None:
            x = x * (x.square().sum(-1, keepdim=True) / case["D"] + _EPS).rsqrt() * w.double()
        x = x.transpose(0, 1)
        turned.append(_exact_turn(x, positions, s["frequencies"], case["interleaved"]).transpose(0, 1))
    k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
    k_cache[page, :, slot] = turned[1][token]
    v_cache[page, :, slot] = s["v"].double()[token]
    return [turned[0].contiguous(), k_cache, v_cache]


def _exact_paged(case, s):
    H, Hk, D = case["H"], case["Hk"], case["D"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    token = 0
    for b, (new, n) in enumerate(_lengths(case)):
        at = torch.arange(n, device="cuda")
        page = s["tables"][b].long()[torch.div(at, case["page"], rounding_mode="floor")]
        rows = at[n - new:]
        for h in range(H):
            k, v = (s[name][page, h // (H // Hk), at % case["page"]].double()
                    for name in ("k_cache", "v_cache"))
            out[token:token + new, h] = _exact_rows(
                s["q"][token:token + new, h].double(), k, v, rows, case["window"], case["sinks"],
                torch.ones(n, dtype=torch.bool, device="cuda"), D ** -0.5)[1]
        token += new
    return [out]


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind.startswith("rotary"):
        return _exact_rotary(case, s)
    if kind.startswith("window"):
        return _exact_window(case, s)
    return _exact_append(case, s) if kind == "append" else _exact_paged(case, s)
