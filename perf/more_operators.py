"""What a decoder with rotary positions and bounded attention runs between its pinned linears, as measurable cases.

Five kinds of case: queries and keys are normalised per head and turned to their positions ("rotate"), the
same with the turned keys and the values going into the 4-bit cache in one call ("append"), a chunk of new
tokens attends over the paged cache ("chunk"), and attention that sees a sliding window and a few first
tokens: single or drafted tokens over the cache ("attend") and packed prompts ("prompt").

A row of D dimensions turns by its position p: pair i of the first `rot` dimensions by the angle
p * freqs[i], pairs being (i, i + rot / 2), or (2 i, 2 i + 1) where interleaved; turned dimensions are
multiplied by `magnitude`. A row at position p sees the positions j <= p with j > p - window or j < sinks.

The cache is four tensors: for pages of 64 tokens, H heads of dimension D and blocks of 64
dimensions (NB = D / 64 a row),
  k_hole   u8  [pages, H, 64, D / 2]: the row of a token is [4][NB][8] bytes, byte (c, b, e)
           holding dimensions 64 b + 16 c + 2 e (low nibble) and 64 b + 16 c + 2 e + 1;
  k_absmax f32 [pages, H, NB, 64];
  v_hole   u8  [pages, H, D / 2, 64]: row 16 p + d, column t holds dimensions 32 p + d (low
           nibble) and 32 p + 16 + d of token t;
  v_absmax f32 [pages, H, NB, 64];
and an element stands for PARENT[nibble] * absmax. Head counts and widths are those of this
repository's benchmark (4096 wide with 1024 of keys and values), or generic.
"""
import math

import torch

own = False

PAGE = 64
EPS = 1e-6
_PARENT = (
    -1.0, -0.6961928009986877, -0.5250730514526367, -0.39491748809814453, -0.28444138169288635, -0.18477343022823334,
    -0.09105003625154495, 0.0, 0.07958029955625534, 0.16093020141124725, 0.24611230194568634, 0.33791524171829224,
    0.44070982933044434, 0.5626170039176941, 0.7229568362236023, 1.0)


def listed():
    return [
        # One new token for each of 8 sequences, queries and keys normed: what every layer does at every decode step.
        {"name": "rotate-8", "kind": "rotate", "T": 8, "H": 8, "G": 4, "D": 128, "rot": 128, "interleaved": False, "norm": True, "dtype": "bf16", "far": False},
        # A long prompt's middle, adjacent pairs of half the head turned, positions past the trained length and scaled.
        {"name": "rotate-4095", "kind": "rotate", "T": 4095, "H": 8, "G": 4, "D": 128, "rot": 64, "interleaved": True, "norm": True, "dtype": "bf16", "far": True},
        # The decode step's whole way from its linear to the cache.
        {"name": "append-8", "kind": "append", "T": 8, "H": 8, "G": 4, "D": 128, "rot": 128, "interleaved": False, "norm": False, "dtype": "bf16", "far": False, "skip": 0},
        # A 4096-token prompt's way to the cache.
        {"name": "append-4096", "kind": "append", "T": 4096, "H": 8, "G": 4, "D": 128, "rot": 128, "interleaved": False, "norm": True, "dtype": "bf16", "far": False, "skip": 0},
        # A follow-up of a few words to a long conversation: few rows, many keys.
        {"name": "chunk-16", "kind": "chunk", "B": 1, "L": 8000, "new": 16, "G": 4, "H": 8, "D": 128, "ragged": False, "fresh": False, "window": 0, "sinks": 0},
        # A document's next 512 tokens, which see one another as they were computed and the rest as the cache holds it.
        {"name": "chunk-512", "kind": "chunk", "B": 1, "L": 16384, "new": 512, "G": 4, "H": 8, "D": 128, "ragged": False, "fresh": True, "window": 0, "sinks": 0},
        # Chunks of every length after contexts of every length in one step.
        {"name": "chunk-ragged", "kind": "chunk", "B": 12, "L": 4097, "new": 301, "G": 4, "H": 10, "D": 64, "ragged": True, "fresh": False, "window": 0, "sinks": 0},
        # The largest step of a long document: the matrix cores.
        {"name": "chunk-2048", "kind": "chunk", "B": 1, "L": 16384, "new": 2048, "G": 4, "H": 8, "D": 128, "ragged": False, "fresh": False, "window": 0, "sinks": 0},
        # A decode batch at long context with a window of 1024: its pages in between are given back.
        {"name": "attend-32x8192", "kind": "attend", "B": 32, "L": 8192, "nq": 1, "G": 4, "H": 8, "D": 128, "ragged": False, "window": 1024, "sinks": 4, "dropped": True},
        # Three drafted tokens of requests of every length, a few finished ones among them.
        {"name": "attend-draft3", "kind": "attend", "B": 48, "L": 4097, "nq": 3, "G": 4, "H": 5, "D": 64, "ragged": True, "window": 1000, "sinks": 70, "dropped": False},
        # One long document under a window of 1024 and 4 first tokens.
        {"name": "prompt-8192", "kind": "prompt", "B": 1, "L": 8192, "prefix": 0, "G": 4, "H": 8, "D": 128, "ragged": False, "window": 1024, "sinks": 4},
        # A packed batch of prompts of different lengths, each after keys it already has.
        {"name": "prompt-packed", "kind": "prompt", "B": 12, "L": 701, "prefix": 200, "G": 4, "H": 10, "D": 64, "ragged": True, "window": 130, "sinks": 65},
    ]


def _log(rng, lo, hi, step=1):
    """A size between lo and hi, spread over its logarithm, a multiple of step."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(step, int(round(v / step)) * step)


def draw(rng):
    kind = rng.choice(("rotate", "rotate", "append", "append", "chunk", "chunk", "chunk", "attend", "attend", "prompt", "prompt"))
    D = rng.choice((64, 128, 128))
    if kind in ("rotate", "append"):
        if kind == "rotate":
            D = rng.choice((64, 80, 96, 128, 128, 256))
        case = {"kind": kind, "T": _log(rng, 1, 4096), "H": rng.choice((1, 2, 5, 8)), "G": rng.choice((1, 3, 4, 5)), "D": D,
                "rot": rng.choice((D, D, max(16, D // 32 * 16), 16 * max(1, D // 64))), "interleaved": rng.random() < 0.4,
                "norm": rng.random() < 0.5, "dtype": rng.choice(("bf16", "bf16", "f32")), "far": rng.random() < 0.4}
        return {**case, "skip": rng.choice((0, 0, 3))} if kind == "append" else case
    G, H = rng.choice((1, 3, 4, 8)), rng.choice((1, 2, 4, 8))
    window, sinks = (0, 0) if kind == "chunk" and rng.random() < 0.6 else (_log(rng, 1, 4096), rng.choice((0, 1, 4, 64, 100)))
    if kind == "chunk":
        new = _log(rng, 2, 1024)
        L = _log(rng, 1, 12000)
        most = max(1, min(16, 12000 // L, 1500 // new))
        return {"kind": kind, "B": _log(rng, 1, most), "L": L + new, "new": new, "G": min(G, 32 // H), "H": H, "D": D,
                "ragged": rng.random() < 0.5, "fresh": rng.random() < 0.5, "window": window, "sinks": sinks}
    if kind == "attend":
        L = _log(rng, 1, 16384)
        return {"kind": kind, "B": _log(rng, 1, max(1, min(64, 200000 // L))), "L": L, "nq": rng.choice((1, 1, 1, 2, 5)), "G": G,
                "H": H, "D": D, "ragged": rng.random() < 0.5, "window": window, "sinks": sinks, "dropped": rng.random() < 0.5}
    L = _log(rng, 1, 6000)
    return {"kind": kind, "B": _log(rng, 1, max(1, min(16, 6000 // L))), "L": L, "prefix": rng.choice((0, 0, _log(rng, 1, 500))), "G": G,
            "H": min(H, 4), "D": D, "ragged": rng.random() < 0.5, "window": window, "sinks": sinks}


def _spread(case, most):
    """One of 1 .. most for each sequence, the same for every seed, all of them `most` where the case is not ragged."""
    if not case["ragged"]:
        return [most] * case["B"]
    return [1 + int((most - 1) * ((0.618034 * (i + 1)) % 1.0)) for i in range(case["B"])]


def _rows(case):
    """(query rows, keys) of each sequence; a ragged batch of the cache's has every sixth length at 0 (a finished request's place)."""
    n = _spread(case, case["L"])
    if case["kind"] == "prompt":
        return n, [x + case["prefix"] for x in n]
    if case["kind"] == "attend":
        return [case["nq"]] * case["B"], [0 if case["ragged"] and i % 6 == 5 else x for i, x in enumerate(n)]
    new = _spread(case, case["new"])[::-1]
    return new, [max(x, y) for x, y in zip(n, new)]


def _starts(lengths):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return at


def _plan(case):
    """What says how rows turn: base 500000 and, for far positions, the slow half scaled by parts for 8 times the trained 8192."""
    return {"base": 500000.0, "factor": 8.0, "trained": 8192, "slow": 1.0, "fast": 4.0} if case["far"] else {"base": 10000.0}


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) % (1 << 62))


def _randn(g, *shape):
    return torch.randn(shape, device="cuda", generator=g)


def _parent():
    return torch.tensor(_PARENT, device="cuda")


def _int32(v):
    return torch.tensor(v, device="cuda", dtype=torch.int32)


def _nibbles(g, *shape):
    """Packed bytes with the code frequencies that normal values under a block-64 absmax have."""
    par = _parent()
    edges = (par[1:] + par[:-1]) / 2
    v = torch.randn((2, *shape), device="cuda", generator=g).mul_(0.4).clamp_(-1, 1)
    c = torch.bucketize(v, edges, out_int32=True)
    return (c[0] | (c[1] << 4)).to(torch.uint8)


def _cache(g, pages, H, D):
    nb = D // 64
    amax = lambda: torch.rand((pages, H, nb, PAGE), device="cuda", generator=g).mul_(2).add_(1.5)  # noqa: E731
    return (_nibbles(g, pages, H, PAGE, D // 2), amax(), _nibbles(g, pages, H, D // 2, PAGE), amax())


def prepare(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    s = dict(case)
    H, G, D = case["H"], case["G"], case["D"]
    if kind in ("rotate", "append"):
        T = case["T"]
        dt = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
        # what the linear gives: a token's queries, keys and values side by side; keys have a few large channels
        qkv = _randn(g, T, (G + 2) * H, D)
        qkv[:, G * H:(G + 1) * H] *= 1 + 4 * (torch.rand(D, device="cuda", generator=g) < 0.05)
        s["qkv"] = qkv.to(dt)
        # a prompt's tokens follow each other, a decode batch's stand anywhere
        if T >= 64:
            s["pos"] = torch.arange(T, device="cuda") + (20000 if case["far"] else 0)
        else:
            s["pos"] = torch.randint(0, 1 << 20 if case["far"] else 8192, (T,), device="cuda", generator=g)
        for name in ("q_norm", "k_norm"):
            s[name] = (1 + 0.2 * _randn(g, D)).to(dt) if case["norm"] else None
        plan = _plan(case)
        s["freqs"] = _freqs(case["rot"], **plan).cuda()
        s["magnitude"] = 0.1 * math.log(plan["factor"]) + 1 if case["far"] else 1.0
        if kind == "append":
            pages = (T + PAGE - 1) // PAGE + 4
            order = torch.randperm(pages, device="cuda", generator=g)
            at = torch.arange(T, device="cuda") + int(torch.randint(0, PAGE, (1,), generator=g, device="cuda"))
            slots = order[at // PAGE] * PAGE + at % PAGE
            if case["skip"]:  # places of a padded batch that hold no token
                slots = torch.where(torch.arange(T, device="cuda") % case["skip"] == 1, torch.full_like(slots, -1), slots)
            s["slots"] = slots
            s["cache"] = _cache(g, pages, H, D)
        return s
    n, m = _rows(case)
    s["most"] = max(n)
    s["q"] = _randn(g, sum(n), H * G, D).to(torch.bfloat16)
    s["cu_q"] = _int32(_starts(n))
    if kind == "prompt":
        s["cu_k"] = _int32(_starts(m))
        s["k"], s["v"] = (_randn(g, sum(m), H, D).to(torch.bfloat16) for _ in range(2))
        return s
    B = case["B"]
    wide = max(1, max((x + PAGE - 1) // PAGE for x in m))
    pages = B * wide + 3
    s["cache"] = _cache(g, pages, H, D)
    s["lens"] = _int32(m)
    s["table"] = torch.randperm(pages, device="cuda", generator=g)[: B * wide].view(B, wide).to(torch.int32)
    if case.get("dropped"):  # pages that no row can see any more are the pool's again
        first = torch.arange(wide, device="cuda") * PAGE
        low = s["lens"][:, None] - case["nq"] - case["window"]
        s["table"].masked_fill_((first >= case["sinks"]) & (first + PAGE - 1 <= low), -1)
    if case.get("fresh"):
        s["k"], s["v"] = (_randn(g, sum(n), H, D).to(torch.bfloat16) for _ in range(2))
    return s


def _freqs(rot, base, factor=1.0, trained=0, slow=1.0, fast=4.0):
    """Radians a position, in 64 bits on the host: base^(-2 i / rot), those that turn less than `slow` times in
    the trained length divided by `factor`, those that turn `fast` times kept, in between a mix."""
    f = torch.tensor([base ** (-2.0 * i / rot) for i in range(rot // 2)], dtype=torch.float64)
    if trained:
        keep = ((trained * f / (2 * math.pi) - slow) / (fast - slow)).clamp(0, 1)
        f = f * keep + f / factor * (1 - keep)
    return f


# ------------------------------------------------------------------ one pass
def run(state):
    kind = state["kind"]
    if own:
        from glint_amd import glint_hip
        s, bounds = state, {"window": state.get("window") or None, "sinks": state.get("sinks", 0)}
        if kind in ("rotate", "append"):
            q, k, v = s["qkv"].split([s["H"] * s["G"], s["H"], s["H"]], 1)
            how = {"interleaved": s["interleaved"], "magnitude": s["magnitude"], "q_norm": s["q_norm"], "k_norm": s["k_norm"], "eps": EPS}
            if kind == "rotate":
                return glint_hip.rotate_qk(q, k, s["pos"], s["freqs"], **how)
            turned = glint_hip.kv4_append_rotated(q, k, v, s["pos"], s["freqs"], s["slots"], s["cache"], **how)
            return (turned, *glint_hip.kv4_gather(s["slots"], s["cache"]))
        if kind == "chunk":
            return glint_hip.kv4_attend_chunk(s["q"], s["cache"], s["table"], s["lens"], s["cu_q"], max_q=s["most"], k=s.get("k"),
                                              v=s.get("v"), **bounds)
        if kind == "attend":
            return glint_hip.kv4_attend(s["q"], s["cache"], s["table"], s["lens"], max_q=s["nq"], **bounds)
        return glint_hip.attend_prompt(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], max_q=s["most"], **bounds)
    return {"rotate": _rotate, "append": _append, "chunk": _over_cache, "attend": _over_cache, "prompt": _prompt}[kind](state)


# ------------------------------------------------------------------ the plain forms
def _turned(s, x, norm):
    """[T, heads, D] normed by its own mean square and turned to its positions, in 32 bits (angles in 64)."""
    rot = s["rot"]
    y = x.float()
    if norm is not None:
        y = y * (y.square().mean(-1, keepdim=True) + EPS).rsqrt() * norm.float()
    angle = s["pos"].double()[:, None, None] * s["freqs"]
    c, w = (angle.cos() * s["magnitude"]).float(), (angle.sin() * s["magnitude"]).float()
    if s["interleaved"]:
        a, b = y[..., 0:rot:2], y[..., 1:rot:2]
        front = torch.stack((a * c - b * w, b * c + a * w), -1).flatten(-2)
    else:
        a, b = y[..., :rot // 2], y[..., rot // 2:rot]
        front = torch.cat((a * c - b * w, b * c + a * w), -1)
    return torch.cat((front, y[..., rot:]), -1).to(x.dtype)


def _rotate(s):
    q, k, _ = s["qkv"].split([s["H"] * s["G"], s["H"], s["H"]], 1)
    return _turned(s, q, s["q_norm"]), _turned(s, k, s["k_norm"])


def _k_values(hole, absmax):
    """[..., 64, D / 2] bytes and [..., NB, 64] scales -> f32 [..., 64, D]"""
    nb = absmax.shape[-2]
    b = hole.unflatten(-1, (4, nb, 8))
    code = torch.stack((b & 15, b >> 4), -1).flatten(-2)  # [..., 64, 4, NB, 16]
    val = _parent()[code.int()].transpose(-3, -2).flatten(-2)  # [..., 64, NB, 64]
    return (val * absmax.transpose(-1, -2)[..., None]).flatten(-2)


def _v_values(hole, absmax):
    """[..., D / 2, 64] bytes and [..., NB, 64] scales -> f32 [..., 64, D]"""
    nb = absmax.shape[-2]
    b = hole.unflatten(-2, (2 * nb, 16))
    code = torch.stack((b & 15, b >> 4), -3).flatten(-4, -2)  # [..., D, 64]
    val = _parent()[code.int()].unflatten(-2, (nb, 64)) * absmax[..., None, :]
    return val.flatten(-3, -2).transpose(-1, -2)


def _codes(w):
    """[T, H, D] -> (codes [T, H, NB, 64], absmax [T, H, NB]), the format's rule in 32 bits"""
    w = w.float().unflatten(-1, (-1, 64))
    s = w.abs().amax(-1)
    v = torch.where(s[..., None] == 0, torch.zeros_like(w), w / s[..., None])
    return ((v[..., None] - _parent()).abs().argmin(-1)).to(torch.uint8), s


def _append(s):
    q, k, v = s["qkv"].split([s["H"] * s["G"], s["H"], s["H"]], 1)
    q, k = _turned(s, q, s["q_norm"]), _turned(s, k, s["k_norm"])
    k_hole, k_absmax, v_hole, v_absmax = s["cache"]
    used = s["slots"] >= 0
    slots = s["slots"][used]
    page, at = slots // PAGE, slots % PAGE
    c, a = _codes(k[used])
    c = c.unflatten(-1, (4, 8, 2)).transpose(2, 3)  # [T, H, 4, NB, 8, 2]
    k_hole[page, :, at] = (c[..., 0] | (c[..., 1] << 4)).flatten(2)
    k_absmax[page, :, :, at] = a
    c, a = _codes(v[used])
    c = c.flatten(2).unflatten(-1, (-1, 2, 16))  # [T, H, D / 32, 2, 16]
    v_hole[page, :, :, at] = (c[..., 0, :] | (c[..., 1, :] << 4)).flatten(2)
    v_absmax[page, :, :, at] = a
    slots = s["slots"].clamp(min=0)
    page, at = slots // PAGE, slots % PAGE
    k = _k_values(k_hole[page, :, at][:, :, None], k_absmax[page, :, :, at][..., None])[:, :, 0]
    v = _v_values(v_hole[page, :, :, at][..., None], v_absmax[page, :, :, at][..., None])[:, :, 0]
    keep = used[:, None, None]
    return q, torch.where(keep, k, 0).to(torch.bfloat16), torch.where(keep, v, 0).to(torch.bfloat16)


def _softmax_product(scores, seen, v):
    """softmax over the last axis of what is seen, times v; rows that see nothing give 0"""
    scores = scores.masked_fill(~seen, -math.inf)
    p = (scores - scores.amax(-1, keepdim=True).clamp(min=-3e38)).exp()
    total = p.sum(-1, keepdim=True)
    return (p @ v) / torch.where(total == 0, torch.ones_like(total), total)


def _seen(s, j, last):
    """Whether a row whose own position is `last` sees position j."""
    seen = j <= last
    return seen & ((j > last - s["window"]) | (j < s["sinks"])) if s["window"] else seen


def _over_cache(s):
    k_hole, k_absmax, v_hole, v_absmax = s["cache"]
    H, G, D, nq, B = s["H"], s["G"], s["D"], s["most"], s["B"]
    t = s["table"].long().clamp(min=0)
    k = _k_values(k_hole[t], k_absmax[t]).transpose(1, 2).flatten(2, 3)  # [B, H, tokens, D]
    v = _v_values(v_hole[t], v_absmax[t]).transpose(1, 2).flatten(2, 3)
    cu = s["cu_q"].long()
    n = cu[1:] - cu[:-1]
    row = torch.arange(nq, device="cuda")
    live = row < n[:, None]  # [B, nq]
    last = s["lens"][:, None] - n[:, None] + row
    at = (cu[:-1, None] + row).clamp(max=s["q"].shape[0] - 1)
    if s.get("fresh"):
        b = torch.arange(B, device="cuda")[:, None].expand(B, nq)[live]
        k[b, :, last[live]] = s["k"].float()
        v[b, :, last[live]] = s["v"].float()
    q = s["q"].float()[at].unflatten(2, (H, G)).permute(0, 2, 3, 1, 4).reshape(B, H, G * nq, D)
    scores = (q @ k.transpose(-1, -2)) * D ** -0.5
    seen = _seen(s, torch.arange(k.shape[2], device="cuda"), last[..., None])
    if s.get("dropped"):
        seen &= (s["table"] >= 0).repeat_interleave(PAGE, 1)[:, None]
    o = _softmax_product(scores, seen[:, None, None].expand(B, 1, G, nq, -1).reshape(B, 1, G * nq, -1), v)
    return o.view(B, H, G, nq, D).permute(0, 3, 1, 2, 4).reshape(B, nq, H * G, D)[live].to(torch.bfloat16)


def _prompt(s):
    q, k, v, cu_q, cu_k = s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"]
    H, G, D = s["H"], s["G"], s["D"]
    i, j = torch.arange(q.shape[0], device="cuda"), torch.arange(k.shape[0], device="cuda")
    bi = torch.bucketize(i, cu_q[1:], right=True)
    bj = torch.bucketize(j, cu_k[1:], right=True)
    last = i - cu_q[bi + 1] + cu_k[bi + 1] - cu_k[bi]  # the last key of its sequence that query i sees
    seen = (bi[:, None] == bj) & _seen(s, j - cu_k[bj], last[:, None])
    qh = q.float().view(-1, H, G, D).permute(1, 2, 0, 3)
    scores = (qh @ k.float().permute(1, 2, 0)[:, None]) * D ** -0.5
    o = _softmax_product(scores, seen, v.float().transpose(0, 1)[:, None])
    return o.permute(2, 0, 1, 3).reshape(-1, H * G, D).to(torch.bfloat16)


# ------------------------------------------------------------------ bytes and operations
def work(case):
    kind, H, G, D = case["kind"], case["H"], case["G"], case["D"]
    size = 2 if case.get("dtype", "bf16") == "bf16" else 4
    held = D // 2 + 4 * (D // 64)  # bytes of one key or value in the cache
    if kind in ("rotate", "append"):
        T = case["T"]
        turned = T * (G + 1) * H * D
        flops = 6 * T * (G + 1) * H * case["rot"] // 2 + (4 * turned if case["norm"] else 0)
        if kind == "rotate":
            return {"bytes": 2 * turned * size + 8 * T, "flops": flops}
        into = T * (G + 2) * H * D * size + T * G * H * D * size + 2 * T * H * held + 16 * T
        return {"bytes": into + 2 * T * H * (held + 2 * D), "flops": flops + 16 * T * H * D}
    n, m = _rows(case)
    pairs = keys = 0
    for x, y in zip(n, m):
        seen = [_count(case, y - x + i) for i in range(x)]
        pairs += sum(seen)
        low = max(0, y - x - (case["window"] or y) + 1)  # the window of the first row
        keys += y - max(0, low - case["sinks"]) if y > 0 else 0
    rows = sum(n) * H * G * D * 4
    flops = 4 * H * G * D * pairs
    if kind == "prompt":
        return {"bytes": rows + keys * H * D * 4, "flops": flops}
    fresh = sum(n) if case.get("fresh") else 0
    return {"bytes": rows + (keys - fresh) * H * 2 * held + fresh * H * D * 4, "flops": flops}


def _count(case, last):
    """How many positions a row at `last` sees."""
    if last < 0:
        return 0
    if not case["window"]:
        return last + 1
    low = max(0, last - case["window"] + 1)
    return last + 1 - low + min(low, case["sinks"])


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    par = torch.tensor(_PARENT, device="cuda", dtype=torch.float64)
    kind = case["kind"]
    H, G, D = case["H"], case["G"], case["D"]
    if kind in ("rotate", "append"):
        rows = s["qkv"].double()
        q, k = _exact_turn(s, rows[:, :H * G], s["q_norm"]), _exact_turn(s, rows[:, H * G:H * G + H], s["k_norm"])
        if kind == "rotate":
            return q, k
        # the cache takes a key as the call would return it: in the inputs' type
        k = k.to(s["qkv"].dtype).double()
        return q, *(_exact_held(x, s["slots"]) for x in (k, rows[:, H * G + H:]))
    out = torch.zeros(s["q"].shape, device="cuda", dtype=torch.float64)
    q = s["q"].double()
    n, m = _rows(case)
    q_at, k_at = _starts(n), _starts(m)
    for b in range(case["B"]):
        nq, nk = n[b], m[b]
        if nk == 0:
            continue
        if kind == "prompt":
            k, v = (s[x][k_at[b]:k_at[b + 1]].double() for x in ("k", "v"))
        else:
            k, v = _held(s, par, b, nk)
            if case.get("fresh"):
                k[nk - nq:], v[nk - nq:] = (s[x][q_at[b]:q_at[b + 1]].double() for x in ("k", "v"))
        for i in range(0, nq, 2048):
            c = min(2048, nq - i)
            j = torch.arange(nk, device="cuda")[None]
            p = (torch.arange(i, i + c, device="cuda") + (nk - nq))[:, None]
            hidden = j > p
            if case["window"]:
                hidden |= (p - j >= case["window"]) & (j >= case["sinks"])
            rows = slice(q_at[b] + i, q_at[b] + i + c)
            for h in range(H * G):
                z = torch.mm(q[rows, h], k[:, h // G].t().contiguous()) / math.sqrt(D)
                z[hidden] = -math.inf
                w = torch.softmax(z, 1)
                w = torch.where(hidden.all(1)[:, None], 0.0, w)
                out[rows, h] = torch.mm(w, v[:, h // G].contiguous())
    return out


def _exact_turn(s, x, norm):
    if norm is not None:
        x = x / torch.sqrt((x * x).sum(2, keepdim=True) / x.shape[2] + EPS) * norm.double()
    x = x.clone()
    angle = torch.outer(s["pos"].double(), s["freqs"])
    turn = torch.polar(torch.full_like(angle, s["magnitude"]), angle)[:, None]
    i = torch.arange(s["rot"] // 2, device="cuda")
    first, second = (2 * i, 2 * i + 1) if s["interleaved"] else (i, i + s["rot"] // 2)
    z = torch.complex(x[..., first], x[..., second]) * turn
    x[..., first], x[..., second] = z.real, z.imag
    return x


def _exact_held(x, slots):
    """What the cache holds of rows x: the nearest of the 16 values, times the block's largest magnitude."""
    rows = x.reshape(-1, 64)
    top = rows.abs().max(1).values
    best = torch.full_like(rows, math.inf)
    held = torch.zeros_like(rows)
    unit = rows / torch.where(top > 0, top, 1.0)[:, None]
    for value in _PARENT:
        d = (unit - value).abs()
        held = torch.where(d < best, value, held)
        best = torch.minimum(best, d)
    held = (held * top[:, None]).view(x.shape)
    held[slots < 0] = 0
    return held


def _held(s, par, b, n):
    """The first n keys and values of sequence b, [n, H, D] in 64 bits, element by element from the layout."""
    k_hole, k_absmax, v_hole, v_absmax = s["cache"]
    t = torch.arange(n, device="cuda")
    page, at = s["table"][b].long()[t // PAGE].clamp(min=0)[:, None, None], (t % PAGE)[:, None, None]
    h = torch.arange(s["H"], device="cuda")[None, :, None]
    d = torch.arange(s["D"], device="cuda")[None, None, :]
    nb = s["D"] // 64
    k = k_hole[page, h, at, ((d % 64) // 16 * nb + d // 64) * 8 + d % 16 // 2].long() >> (4 * (d % 2)) & 15
    v = v_hole[page, h, d // 32 * 16 + d % 16, at].long() >> (4 * (d % 32 // 16)) & 15
    return par[k] * k_absmax[page, h, d // 64, at].double(), par[v] * v_absmax[page, h, d // 64, at].double()
