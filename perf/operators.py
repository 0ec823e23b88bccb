"""Performance cases of the token mixers that stand between a decoder layer's
projections: the gated delta rule of the linear-attention layers, the rotary
positions and the paged key-value cache of the full-attention layers.

A case is a dict of plain values; `listed()` names twelve, `draw(rng)` gives
more of the same ranges.  `prepare` builds what a program holds before the call,
`run` is one pass (`own`: the framework's operators, else their plain form in
32 bits), `exact` the same outputs from the definitions in 64 bits.

Kinds:
  delta_step   gated delta rule, one token for each of B sequences
  delta_chunk  gated delta rule over whole (ragged) sequences, state in and out
  attn         attention of one new token per sequence over a paged cache
  rotary       several-axis rotary positions of q and k
  rotary_cache the same, with the rotated k and the v written into the paged cache
"""
from __future__ import annotations

import math
import sys
from types import SimpleNamespace

import torch

own = False

CHUNK = 64
NORM_EPS = 1e-6
THETA = 1e7


def _pkg():
    name = "minicpmv_amd"
    if name not in sys.modules:
        import __graft_entry__
        __graft_entry__.load_package()
    return sys.modules[name]


# ---------------------------------------------------------------------- cases --
def listed():
    return [
        # a linear-attention layer's share of one decoded token: launch and latency
        {"name": "delta_step_1", "kind": "delta_step", "B": 1, "Hk": 16, "Hv": 16, "D": 128},
        # the same for an odd batch of conversations, each with a state of its own
        {"name": "delta_step_53", "kind": "delta_step", "B": 53, "Hk": 16, "Hv": 16, "D": 128},
        # a short text prompt from an empty state
        {"name": "delta_prompt_77", "kind": "delta_chunk", "B": 1, "T": 77, "Hk": 16, "Hv": 16, "D": 128, "carry": 0},
        # seven prompts of different lengths continued from their states, two value heads to a key head
        {"name": "delta_ragged_2900", "kind": "delta_chunk", "B": 7, "T": 2900, "Hk": 16, "Hv": 32, "D": 128, "carry": 1},
        # one long multi-image prompt
        {"name": "delta_long_8192", "kind": "delta_chunk", "B": 1, "T": 8192, "Hk": 16, "Hv": 16, "D": 128, "carry": 1},
        # a full-attention layer's share of one decoded token after an image and a question
        {"name": "attn_1x1100", "kind": "attn", "B": 1, "len": 1100, "Hq": 8, "Hkv": 2, "D": 256, "page": 16},
        # a batch of conversations of very different lengths, one slot of it empty
        {"name": "attn_41x4096", "kind": "attn", "B": 41, "len": 4096, "Hq": 8, "Hkv": 2, "D": 256, "page": 32},
        # one very long context
        {"name": "attn_1x200000", "kind": "attn", "B": 1, "len": 200000, "Hq": 8, "Hkv": 2, "D": 256, "page": 64},
        # narrower heads, more of them
        {"name": "attn_16x2000_d128", "kind": "attn", "B": 16, "len": 2000, "Hq": 32, "Hkv": 8, "D": 128, "page": 16},
        # one decoded token's q, k and v
        {"name": "rotary_cache_1", "kind": "rotary_cache", "T": 1, "Hq": 8, "Hkv": 2, "D": 256, "rot": 64, "page": 16},
        # an image's tokens with a question, the whole head rotated
        {"name": "rotary_1100", "kind": "rotary", "T": 1100, "Hq": 16, "Hkv": 4, "D": 128, "rot": 128, "mixed": 0},
        # a long multi-image prompt into the cache
        {"name": "rotary_cache_8192", "kind": "rotary_cache", "T": 8192, "Hq": 8, "Hkv": 2, "D": 256, "rot": 64, "page": 32},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("delta_step", "delta_chunk", "delta_chunk", "attn", "attn", "rotary", "rotary_cache"))
    case = {"kind": kind}
    if kind.startswith("delta"):
        hk = rng.choice((2, 4, 8, 16))
        hv = hk * rng.choice((1, 1, 2))
        d = rng.choice((64, 128, 128))
        case.update(Hk=hk, Hv=hv, D=d)
        if kind == "delta_step":
            case["B"] = _log_int(rng, 1, 53 * 16 // hv)
        else:
            T = _log_int(rng, 1, 8192 * 16 // max(hv, 16))
            case.update(T=T, B=rng.randint(1, min(9, T)), carry=rng.randrange(2))
    elif kind == "attn":
        hq, hkv, d = rng.choice(((8, 2, 256), (8, 2, 256), (32, 8, 128), (16, 16, 64), (12, 1, 128)))
        b = _log_int(rng, 1, 64)
        case.update(B=b, len=_log_int(rng, 1, 200000 * 512 // (b * hkv * d)), Hq=hq, Hkv=hkv, D=d,
                    page=rng.choice((16, 32, 64, 128)))
    else:
        hq, hkv, d, rot = rng.choice(((8, 2, 256, 64), (8, 2, 256, 64), (16, 4, 128, 128), (16, 16, 64, 64)))
        case.update(T=_log_int(rng, 1, 8192), Hq=hq, Hkv=hkv, D=d, rot=rot)
        if kind == "rotary":
            case["mixed"] = rng.randrange(2)
        else:
            case["page"] = rng.choice((16, 32, 64, 128))
    return case


# --------------------------------------------------------------------- inputs --
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 2654435761 % (1 << 62))


def _randn(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * std


def _rand(g, *shape):
    return torch.rand(*shape, generator=g, device="cuda", dtype=torch.float32)


def _lengths(g, B, T):
    """B lengths of at least one token that add up to T."""
    cuts = (torch.randperm(T - 1, generator=g, device="cuda")[: B - 1] + 1).sort().values.tolist()
    edges = [0, *cuts, T]
    return [b - a for a, b in zip(edges, edges[1:])]


def _delta_inputs(case, g):
    """q, k and v as columns of one projection's output (their rows are strided), the
    gates of a softplus decay with its own rate per head and of a sigmoid."""
    Hk, Hv, D = case["Hk"], case["Hv"], case["D"]
    step = case["kind"] == "delta_step"
    n = case["B"] if step else case["T"]
    qkv = _randn(g, n, (2 * Hk + Hv) * D)
    qkv[:, Hk * D:2 * Hk * D] += 0.5 * _randn(g, 1, Hk * D)      # keys of one head lean the same way
    qkv = (qkv * torch.sigmoid(qkv)).half()                      # behind a convolution and its silu
    s = SimpleNamespace()
    s.q = qkv[:, :Hk * D].view(n, Hk, D)
    s.k = qkv[:, Hk * D:2 * Hk * D].view(n, Hk, D)
    s.v = qkv[:, 2 * Hk * D:].view(n, Hv, D)
    rate = torch.exp(math.log(0.05) + _rand(g, Hv) * math.log(16 / 0.05))
    s.g = -rate * torch.nn.functional.softplus(_randn(g, n, Hv) - 3.0)
    s.beta = torch.sigmoid(_randn(g, n, Hv))
    s.lens = [1] * n if step else _lengths(g, case["B"], n)
    s.cu = torch.tensor([0, *torch.tensor(s.lens).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    s.state = _randn(g, case["B"], Hv, D, D, std=0.2) if case.get("carry", 1) else None
    s.scale = D ** -0.5
    return s


def _spread(case):
    """The sequences' lengths: the longest, an empty slot, and between them few long ones, many short ones."""
    B, L = case["B"], case["len"]
    return [L] if B == 1 else [L, 0, *(max(1, int(L * ((i + 0.5) / (B - 2)) ** 2)) for i in range(B - 2))]


def _attn_inputs(case, g):
    """A pool of pages in shuffled order.  What a page holds after its sequence's end, and
    every page that no sequence owns, is left over from earlier use: NaN here."""
    B, L, Hq, Hkv, D, P = (case[n] for n in ("B", "len", "Hq", "Hkv", "D", "page"))
    s = SimpleNamespace(max_len=L)
    lens = [_spread(case)[i] for i in torch.randperm(B, generator=g, device="cuda").tolist()]
    width = -(-L // P)
    used = sum(-(-n // P) for n in lens)
    pool = used + 3
    order = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(B, width, dtype=torch.int32, device="cuda")
    s.k = torch.full((pool, P, Hkv, D), math.nan, dtype=torch.float16, device="cuda")
    s.v = torch.full_like(s.k, math.nan)
    at = 0
    for b, n in enumerate(lens):
        m = -(-n // P)
        own_pages = order[at:at + m]
        table[b, :m] = own_pages
        at += m
        if n:
            for pool_t in (s.k, s.v):
                rows = torch.full((m * P, Hkv, D), math.nan, dtype=torch.float16, device="cuda")
                rows[:n] = _randn(g, n, Hkv, D).half()
                pool_t[own_pages.long()] = rows.view(m, P, Hkv, D)
    s.q = (_randn(g, B, Hq, D) * 2.0).half()
    s.table, s.lens = table, torch.tensor(lens, dtype=torch.int32, device="cuda")
    s.scale = D ** -0.5
    return s


def _positions(g, T):
    """Time, height and width of a prompt: text, where the three run together, with images
    between, whose tokens share one time and lie on a grid; far into a conversation."""
    start = int(torch.randint(0, 200000, (1,), generator=g, device="cuda"))
    pos, t, left = [], start, T
    while left > 0:
        n = min(left, int(torch.randint(1, 120, (1,), generator=g, device="cuda")))
        pos += [(t + i, t + i, t + i) for i in range(n)]
        t, left = t + n, left - n
        h, w = (int(x) for x in torch.randint(4, 32, (2,), generator=g, device="cuda"))
        n = min(left, h * w)
        pos += [(t, t + i // w, t + i % w) for i in range(n)]
        t, left = t + max(h, w), left - n
    return torch.tensor(pos, dtype=torch.int64, device="cuda").t().contiguous()


def _rotary_inputs(case, g):
    """q, k and v as columns of one projection's output; the frequencies and the axis each goes by."""
    T, Hq, Hkv, D, rot = (case[n] for n in ("T", "Hq", "Hkv", "D", "rot"))
    s = SimpleNamespace()
    qkv = _randn(g, T, (Hq + 2 * Hkv) * D).half()
    s.q = qkv[:, :Hq * D].view(T, Hq, D)
    s.k = qkv[:, Hq * D:(Hq + Hkv) * D].view(T, Hkv, D)
    s.v = qkv[:, (Hq + Hkv) * D:].view(T, Hkv, D)
    s.pos = _positions(g, T)
    half = rot // 2
    i = torch.arange(half, device="cuda")
    s.freq = THETA ** (-i.double() / half)
    side = half * 5 // 16                                        # height's and width's share; time has the rest
    if case.get("mixed", 1):                                     # the axes take turns: t h w t h w ... t t
        s.axis = torch.where((i % 3 == 1) & (i < 3 * side), 1, torch.where((i % 3 == 2) & (i < 3 * side), 2, 0)).int()
    else:                                                        # one after the other: t ... h ... w ...
        s.axis = torch.where(i < half - 2 * side, 0, torch.where(i < half - side, 1, 2)).int()
    if case["kind"] == "rotary_cache":
        P = case["page"]
        pages = -(-T // P) + 2
        order = torch.randperm(pages, generator=g, device="cuda")
        at = torch.arange(T, device="cuda")
        s.slots = order[at // P] * P + at % P
        s.kc = torch.zeros(pages, P, Hkv, D, dtype=torch.float16, device="cuda")
        s.vc = torch.zeros_like(s.kc)
    return s


def _inputs(case, seed):
    make = _delta_inputs if case["kind"].startswith("delta") else _attn_inputs if case["kind"] == "attn" else _rotary_inputs
    return make(case, _gen(seed))


def prepare(case, seed):
    s = _inputs(case, seed)
    s.case, s.kind = case, case["kind"]
    if s.kind.startswith("delta"):
        s.out = torch.empty(s.v.shape, dtype=torch.float16, device="cuda")
        s.state_out = torch.empty(case["B"], case["Hv"], case["D"], case["D"], dtype=torch.float32, device="cuda")
        s.index = _padded(s.lens) if s.kind == "delta_chunk" else None
    else:
        s.q_out = torch.empty(s.q.shape, dtype=torch.float16, device="cuda")
        if s.kind == "rotary":
            s.k_out = torch.empty(s.k.shape, dtype=torch.float16, device="cuda")
    return s


# ---------------------------------------------------------------- plain forms --
def _padded(lens):
    """Where the rows of [sequences, chunks, CHUNK] lie in the packed tokens (one past the
    last: an empty row), and where the tokens lie there."""
    n, chunks = sum(lens), -(-max(lens) // CHUNK)
    rows = torch.full((len(lens), chunks * CHUNK), n, dtype=torch.int64)
    at = 0
    for b, m in enumerate(lens):
        rows[b, :m] = torch.arange(at, at + m)
        at += m
    rows = rows.cuda()
    place = torch.empty(n + 1, dtype=torch.int64, device="cuda")
    place[rows.flatten()] = torch.arange(rows.numel(), device="cuda")
    return rows, place[:n]


def _unit(x):
    return x * torch.rsqrt(x.square().sum(-1, keepdim=True) + NORM_EPS)


def _plain_step(s):
    r = s.v.shape[1] // s.k.shape[1]
    q = (_unit(s.q.float()) * s.scale).repeat_interleave(r, 1)
    k = _unit(s.k.float()).repeat_interleave(r, 1)
    S = s.state * torch.exp(s.g)[..., None, None]
    u = (s.v.float() - (k[..., None] * S).sum(-2)) * s.beta[..., None]
    S = S + k[..., None] * u[..., None, :]
    return (q[..., None] * S).sum(-2).half(), S


def _plain_chunk(s):
    """The rule over chunks of 64 tokens.  Inside one, with G the running sum of g, the
    corrected values solve (I + L) U = beta (V - e^G K S), L[i, j] = beta_i e^(G_i - G_j)
    k_i . k_j below the diagonal; all chunks' inverses are built at once, row by row."""
    rows, place = s.index
    r = s.v.shape[1] // s.k.shape[1]
    Hv, D = s.v.shape[1:]
    B, nc = rows.shape[0], rows.shape[1] // CHUNK

    def chunks(x):                                               # [n, H, ...] -> [B, H, chunks, CHUNK, ...]
        x = torch.cat((x, torch.zeros_like(x[:1])))[rows.flatten()]
        return x.view(B, nc, CHUNK, *x.shape[1:]).movedim(3, 1)

    q = chunks((_unit(s.q.float()) * s.scale).repeat_interleave(r, 1))
    k = chunks(_unit(s.k.float()).repeat_interleave(r, 1))
    v, g, beta = chunks(s.v.float()), chunks(s.g), chunks(s.beta)
    G = g.double().cumsum(-1)
    i = torch.arange(CHUNK, device="cuda")
    low = i[:, None] >= i
    fall = torch.exp(torch.where(low, G[..., :, None] - G[..., None, :], -math.inf).float())
    kt = k.transpose(-1, -2).contiguous()
    A = (k @ kt) * fall * beta[..., None] * (i[:, None] > i)
    inv = torch.eye(CHUNK, device="cuda").expand_as(A).contiguous()
    for j in range(1, CHUNK):
        inv[..., j, :j] = -(A[..., j, :j, None] * inv[..., :j, :j]).sum(-2)
    eG = torch.exp(G).float()[..., None]
    W = inv @ (k * eG * beta[..., None])
    V = inv @ (v * beta[..., None])
    P = (q @ kt) * fall
    qe = q * eG
    keep = torch.exp(G[..., -1:]).float()[..., None]
    ke = (k * torch.exp(G[..., -1:] - G).float()[..., None]).transpose(-1, -2).contiguous()
    S = torch.zeros(B, Hv, D, D, device="cuda") if s.state is None else s.state
    out = torch.empty(B, Hv, nc, CHUNK, D, device="cuda")
    for c in range(nc):                                          # rows past a sequence's end change nothing: k = v = g = 0
        U = V[:, :, c] - W[:, :, c] @ S
        out[:, :, c] = qe[:, :, c] @ S + P[:, :, c] @ U
        S = S * keep[:, :, c] + ke[:, :, c] @ U
    return out.movedim(1, 3).reshape(-1, Hv, D)[place].half(), S


def _plain_attn(s):
    B, Hq, D = s.q.shape
    P, Hkv = s.k.shape[1:3]
    live = torch.arange(s.table.shape[1] * P, device="cuda") < s.lens[:, None]          # [B, len]
    kv = [torch.where(live[..., None, None], t[s.table.long()].flatten(1, 2), 0).float().transpose(1, 2).contiguous()
          for t in (s.k, s.v)]                                                          # [B, Hkv, len, D]
    q = s.q.float().view(B, Hkv, Hq // Hkv, D) * s.scale
    w = q @ kv[0].transpose(-1, -2).contiguous()
    w = torch.where(live[:, None, None], w, -math.inf)
    w = torch.exp(w - w.amax(-1, keepdim=True).clamp_min(-3e38))
    total = w.sum(-1, keepdim=True)
    return ((w @ kv[1]) / torch.where(total > 0, total, 1)).view(B, Hq, D).half()


def _turn(x, c, s):
    half = c.shape[-1]
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat((a * c - b * s, b * c + a * s, x[..., 2 * half:]), -1)


def _plain_rotary(s):
    angle = s.pos.t()[:, s.axis.long()].double() * s.freq        # [T, rot / 2]: far positions need 64 bits
    c, sn = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    q, k = _turn(s.q.float(), c, sn).half(), _turn(s.k.float(), c, sn).half()
    if s.kind == "rotary":
        return q, k
    s.kc.flatten(0, 1)[s.slots] = k
    s.vc.flatten(0, 1)[s.slots] = s.v
    return q, s.kc, s.vc


# ------------------------------------------------------------------------ run --
def run(state):
    s = state
    if not own:
        return {"delta_step": _plain_step, "delta_chunk": _plain_chunk, "attn": _plain_attn}.get(s.kind, _plain_rotary)(s)
    pkg = _pkg()
    if s.kind == "delta_step":
        return pkg.gated_delta_rule_step(s.q, s.k, s.v, s.g, s.beta, s.state, scale=s.scale, normalize=True, out=s.out,
                                         state_out=s.state_out)
    if s.kind == "delta_chunk":
        return pkg.gated_delta_rule(s.q, s.k, s.v, s.g, s.beta, s.state, cu_seqlens=s.cu, scale=s.scale, normalize=True,
                                    out=s.out, state_out=s.state_out)
    if s.kind == "attn":
        return pkg.paged_attention_decode(s.q, s.k, s.v, s.table, s.lens, scale=s.scale, max_seq_len=s.max_len, out=s.q_out)
    if s.kind == "rotary":
        return pkg.rotary_axes(s.q, s.k, s.pos, s.freq, s.axis, q_out=s.q_out, k_out=s.k_out)
    pkg.rotary_axes_cached(s.q, s.k, s.v, s.pos, s.freq, s.axis, s.kc, s.vc, s.slots, q_out=s.q_out)
    return s.q_out, s.kc, s.vc


# ------------------------------------------------------------------- measures --
def work(case):
    kind = case["kind"]
    if kind.startswith("delta"):
        Hk, Hv, D, B = (case[n] for n in ("Hk", "Hv", "D", "B"))
        n = case.get("T", B)
        state = 4 * B * Hv * D * D * (1 + case.get("carry", 1))
        # per token and head: k . S, the rank-one update and q . S
        return {"bytes": n * (2 * (2 * Hk + 2 * Hv) * D + 8 * Hv) + state, "flops": 6 * n * Hv * D * D}
    if kind == "attn":
        B, Hq, Hkv, D = (case[n] for n in ("B", "Hq", "Hkv", "D"))
        lens = _spread(case)
        pages = sum(-(-n // case["page"]) for n in lens)
        return {"bytes": 4 * sum(lens) * Hkv * D + 4 * B * Hq * D + 4 * pages + 4 * B, "flops": 4 * sum(lens) * Hq * D}
    T, Hq, Hkv, D, rot = (case[n] for n in ("T", "Hq", "Hkv", "D", "rot"))
    cached = kind == "rotary_cache"
    return {"bytes": T * (4 * (Hq + (2 if cached else 1) * Hkv) * D + 24 + 8 * cached) + 6 * rot,
            "flops": 3 * T * (Hq + Hkv) * rot + 40 * T * rot // 2}


# ---------------------------------------------------------------------- exact --
def _exact_delta(s, case):
    """Token by token, every sequence's t-th together."""
    r = case["Hv"] // case["Hk"]
    lens = torch.tensor(s.lens, device="cuda")
    first = s.cu[:-1].long()
    q, k, v, g, beta = (x.double() for x in (s.q, s.k, s.v, s.g, s.beta))
    q, k = (x / (x.pow(2).sum(-1, keepdim=True) + NORM_EPS).sqrt() for x in (q, k))
    q, k = (x.repeat_interleave(r, 1) for x in (q * s.scale, k))
    S = torch.zeros(case["B"], case["Hv"], case["D"], case["D"], dtype=torch.float64, device="cuda")
    if s.state is not None:
        S += s.state
    out = torch.zeros(v.shape, dtype=torch.float64, device="cuda")
    for t in range(max(s.lens)):
        on = (t < lens).nonzero()[:, 0] if min(s.lens) <= t else slice(None)
        at = first[on] + t
        H = S[on] * g[at].exp()[..., None, None]
        d = v[at] - (H * k[at][..., None]).sum(2)
        H = H + k[at][..., None] * (d * beta[at][..., None])[..., None, :]
        out[at] = (H * q[at][..., None]).sum(2)
        S[on] = H
    return out, S


def _exact_attn(s, case):
    Hq, Hkv, P = case["Hq"], case["Hkv"], case["page"]
    out = torch.zeros(s.q.shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(s.lens.tolist()):
        if n == 0:
            continue
        pages = s.table[b, :-(-n // P)].long()
        for h in range(Hkv):
            k, v = (t[pages, :, h].reshape(-1, case["D"])[:n].double() for t in (s.k, s.v))
            heads = slice(h * Hq // Hkv, (h + 1) * Hq // Hkv)
            out[b, heads] = torch.softmax(k @ s.q[b, heads].double().t() * s.scale, 0).t() @ v
    return out


def _exact_rotary(s, case):
    half = case["rot"] // 2
    out = []
    angle = torch.stack([s.pos[int(a)].double() * f for a, f in zip(s.axis.tolist(), s.freq.tolist())], -1)
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    for x in (s.q.double(), s.k.double()):
        z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * turn
        out.append(torch.cat((z.real, z.imag, x[..., 2 * half:]), -1))
    if case["kind"] == "rotary":
        return tuple(out)
    caches = []
    for x in (out[1], s.v.double()):
        flat = torch.zeros(s.kc.shape, dtype=torch.float64, device="cuda").flatten(0, 1)
        flat.index_copy_(0, s.slots, x)
        caches.append(flat.view(s.kc.shape))
    return out[0], caches[0], caches[1]


def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"].startswith("delta"):
        return _exact_delta(s, case)
    return _exact_attn(s, case) if case["kind"] == "attn" else _exact_rotary(s, case)
