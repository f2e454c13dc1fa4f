"""The operators of serving with drafted tokens, by which their speed is followed: keys and values stored in 8 bits and read back, attention of
drafted tokens (single tokens, chains, trees, portions of prompts) over a history, log probabilities of tokens with entropy and alternatives.

``prepare`` makes inputs and caches on the GPU from the seed; ``run`` is one call of a user's program: of the package's operators, or, where
``own`` is false, of their plain form in elementary torch operations; ``exact`` is the same result in 64 bits.
"""
import math
import types

import torch

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
E4M3, U8 = torch.float8_e4m3fn, torch.uint8
CACHE = {"bf16": BF16, "int8": torch.int8, "e4m3": E4M3}
ACT = {"bf16": BF16, "f32": F32}
EPS = 1e-6
LEAST = 2.0 ** -100                 # a vector's largest entry counts as at least that when its scale is chosen

own = False


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # the smallest call: the keys and values of one decoded token of four requests (8 key/value heads of 128 channels)
        {"name": "store_token", "kind": "store", "cache": "e4m3", "act": "bf16", "seqs": 4, "tokens": 1, "past": 1900, "G": 8, "dim": 128, "vdim": 128, "norm": False},
        # four whole prompts of 2048 tokens, values normed per head on their way into the cache (Bebulorn)
        {"name": "store_prompts", "kind": "store", "cache": "e4m3", "act": "bf16", "seqs": 4, "tokens": 2048, "past": 0, "G": 8, "dim": 128, "vdim": 128, "norm": True},
        # portions of odd length of 32-bit activations, stored and read back; key and value heads of different widths
        {"name": "round_ragged", "kind": "round", "cache": "int8", "act": "f32", "seqs": 3, "tokens": 111, "past": 37, "G": 3, "dim": 64, "vdim": 128, "norm": False},
        # whole histories of 16 requests read back as rows, for instance for a kernel that takes bf16 alone
        {"name": "load_histories", "kind": "load", "cache": "int8", "act": "bf16", "seqs": 16, "tokens": 8191, "past": 0, "G": 8, "dim": 128, "vdim": 128, "norm": False},
        # one decoded token of 16 requests over 8-bit histories
        {"name": "attn_token", "kind": "attn", "cache": "int8", "layout": "slots", "seqs": 16, "past": 1901, "spread": 0.0, "tokens": 1, "branch": 0, "H": 16, "G": 8, "dim": 128,
         "vdim": 128, "window": 0, "softcap": 0.0},
        # the headline benchmark's batch with a chain of 8 drafted tokens each (OPT-30B: 56 heads, time-major bf16 cache, 288 positions)
        {"name": "attn_chain_opt", "kind": "attn", "cache": "bf16", "layout": "time", "seqs": 64, "past": 280, "spread": 0.0, "tokens": 8, "branch": 0, "H": 56, "G": 56, "dim": 128,
         "vdim": 128, "window": 0, "softcap": 0.0},
        # trees of 29 drafted tokens behind histories of unequal odd lengths, under a sliding window with capped scores (Bebulorn's attention)
        {"name": "attn_tree_ragged", "kind": "attn", "cache": "e4m3", "layout": "slots", "seqs": 5, "past": 4099, "spread": 0.7, "tokens": 29, "branch": 2, "H": 16, "G": 8, "dim": 128,
         "vdim": 128, "window": 1024, "softcap": 50.0},
        # one request with a very long history and a wide tree of 64 drafted tokens, four query heads to a key head: the largest
        {"name": "attn_tree_long", "kind": "attn", "cache": "int8", "layout": "slots", "seqs": 1, "past": 131003, "spread": 0.0, "tokens": 64, "branch": 3, "H": 32, "G": 8, "dim": 128,
         "vdim": 128, "window": 0, "softcap": 0.0},
        # the next portions of two prompts, of unequal odd lengths, over 8-bit caches
        {"name": "attn_portions", "kind": "attn", "cache": "int8", "layout": "slots", "seqs": 2, "past": 512, "spread": 0.3, "tokens": 1003, "branch": 0, "H": 16, "G": 8, "dim": 128,
         "vdim": 128, "window": 0, "softcap": 0.0},
        # a decoded token of four requests: how likely it was, and five alternatives (OPT's vocabulary)
        {"name": "logprob_token", "kind": "logprob", "act": "f32", "rows": 4, "vocab": 50272, "given": 1, "top": 5, "banned": 0},
        # the tokens of a drafted tree in bf16 over an odd vocabulary with banned ids: three children of each looked up
        {"name": "logprob_tree", "kind": "logprob", "act": "bf16", "rows": 77, "vocab": 50265, "given": 3, "top": 8, "banned": 5},
        # every token of long prompts scored, with twenty alternatives
        {"name": "logprob_prompts", "kind": "logprob", "act": "f32", "rows": 4096, "vocab": 50272, "given": 1, "top": 20, "banned": 0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(("store", "round", "load", "attn", "attn", "attn", "attn", "logprob", "logprob"))
    if kind == "logprob":
        vocab = _log(rng, 500, 100000)
        return {"kind": kind, "act": rng.choice(("bf16", "f32")), "rows": _log(rng, 1, min(4096, 200_000_000 // vocab)), "vocab": vocab, "given": rng.randint(1, 5),
                "top": rng.choice((0, 1, 4, rng.randint(2, 20))), "banned": rng.choice((0, 0, 7))}
    dims = rng.choice(((128, 128), (128, 128), (64, 64), (64, 128), (128, 64)))
    if kind != "attn":
        seqs, G = rng.randint(1, 16), rng.choice((1, 2, 3, 8, 12))
        return {"kind": kind, "cache": rng.choice(("int8", "e4m3")), "act": rng.choice(("bf16", "bf16", "f32")), "seqs": seqs, "tokens": _log(rng, 1, 30000 // (seqs * G) + 1),
                "past": _log(rng, 1, 2000), "G": G, "dim": dims[0], "vdim": dims[1], "norm": rng.random() < 0.4}
    G, rep = rng.choice(((1, 8), (2, 4), (8, 1), (8, 2), (8, 4), (12, 1), (56, 1), (3, 5), (1, 1)))
    H, cache = G * rep, rng.choice(("bf16", "int8", "e4m3"))
    branch = rng.choice((0, 1, 2, 3))
    style = rng.choice(("token", "drafts", "drafts", "drafts", "portions"))
    seqs = _log(rng, 1, 64 if style != "portions" else 4)
    tokens = 1 if style == "token" else _log(rng, 2, 64) if style == "drafts" else _log(rng, 65, 1000)
    past = _log(rng, 1, min(60000, max(8, (1 << 27) // (seqs * max(G * 128, H * tokens // 2)))))
    if style == "portions":
        branch = 0
    return {"kind": kind, "cache": cache, "layout": rng.choice(("slots", "slots", "time")), "seqs": seqs, "past": past, "spread": rng.choice((0.0, 0.5, 0.9)),
            "tokens": tokens, "branch": branch, "H": H, "G": G, "dim": dims[0], "vdim": dims[1], "window": rng.choice((0, 0, _log(rng, 64, 4096))),
            "softcap": rng.choice((0.0, 0.0, 30.0))}


# ------------------------------------------------------------------------------------------------ inputs
def _portions(case):
    """(slot, first position, first row, rows) of every request: slots in an order of their own, histories and portions a little shorter each time."""
    out, row, n = [], 0, case["seqs"]
    for i in range(n):
        less = case.get("spread", 0.0) * i / n
        past = int(case["past"] * (1 - less))
        tokens = max(1, case["tokens"] - (case["tokens"] * i // (3 * n) if case["kind"] != "attn" or case.get("spread") else 0))
        out.append((n - 1 - i, past, row, tokens))
        row += tokens
    return out


def _parents(case, n):
    return [(j - 1) // case["branch"] if j else -1 for j in range(n)]


def _quantise(x, cache, norm):
    """x [rows, heads, dim] in 32 bits -> codes, scales [rows, heads]: the largest magnitude becomes 127, or 224 to 448 by a power of two."""
    if norm:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
    a = x.abs().amax(-1, keepdim=True)
    bad, a = ~torch.isfinite(a), a.clamp(min=LEAST)
    if cache == "int8":
        codes, scale = torch.round(127 * x / a).masked_fill(bad, 0.0).to(torch.int8), a / 127
    else:
        m, e = torch.frexp(a)
        scale = torch.ldexp(torch.ones_like(a), e - 9 + (m > 0.875).to(e.dtype))
        codes = (x / scale).masked_fill(bad, 0.0).to(E4M3)
    return codes, scale.masked_fill(bad, math.nan)[..., 0]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 6007 + 17)

    def rand(*shape, std=1.0, mean=0.0, dtype=BF16):
        return (torch.randn(*shape, generator=g, device="cuda") * std + mean).to(BF16).to(dtype)

    s = types.SimpleNamespace(case=case)
    if case["kind"] == "logprob":
        M, V = case["rows"], case["vocab"]
        x = torch.randn(M, V, generator=g, device="cuda").mul_(2.0)
        likely = torch.randint(0, V, (M, 3), generator=g, device="cuda")          # a few tokens stand out, as they do in a trained model
        x.scatter_add_(1, likely, torch.rand(M, 3, generator=g, device="cuda") * 12.0)
        if case["banned"]:
            x[:, torch.randint(0, V, (case["banned"],), generator=g, device="cuda")] = -math.inf
        s.logits = x.to(ACT[case["act"]])
        s.tokens = torch.randint(0, V, (M, case["given"]), generator=g, device="cuda")
        s.tokens[:, 0] = likely[:, 0]
        return s
    portions = _portions(case)
    n, M = len(portions), portions[-1][2] + portions[-1][3]
    G, dim, vdim, kind = case["G"], case["dim"], case["vdim"], CACHE[case["cache"]]
    cap = max(p[1] + p[3] for p in portions) + 5
    s.segs = torch.tensor(portions, dtype=torch.int32, device="cuda")
    s.M, s.cap, s.max_ctx, s.rows = M, cap, cap - 5, max(p[3] for p in portions)
    if case["kind"] != "attn":
        s.meta = torch.tensor([(a, b + i) for a, b, _, m in portions for i in range(m)], dtype=torch.int32, device="cuda")
        s.k, s.v = rand(M, G * dim, std=1.5, dtype=ACT[case["act"]]), rand(M, G * vdim, std=0.7, dtype=ACT[case["act"]])
        s.slot, s.pos = s.meta[:, 0].long(), s.meta[:, 1].long()
        s.kc, s.vc = (torch.zeros(n, cap, G * d, dtype=U8, device="cuda").view(kind) for d in (dim, vdim))
        s.ks, s.vs = (torch.zeros(n, G, cap, device="cuda") for _ in range(2))
        if case["kind"] == "load":
            for x, d, codes, scales in ((s.k, dim, s.kc, s.ks), (s.v, vdim, s.vc, s.vs)):
                c, a = _quantise(x.float().view(M, G, d), case["cache"], False)
                codes.view(U8)[s.slot, s.pos] = c.view(U8).view(M, G * d)
                scales[s.slot, :, s.pos] = a
        if case["kind"] != "store":
            s.k_out, s.v_out = torch.empty_like(s.k), torch.empty_like(s.v)
        return s
    H = case["H"]
    s.q = rand(M, H * dim, std=1.3)
    s.scale = dim ** -0.5
    s.temp = rand(H, std=0.1, mean=1.0, dtype=F32) if case["softcap"] else None
    s.out = torch.empty(M, H * vdim, dtype=BF16, device="cuda")
    s.row_seg = torch.tensor([i for i, p in enumerate(portions) for _ in range(p[3])], device="cuda")     # of every row: its portion, its place there
    s.row_at = torch.tensor([j for p in portions for j in range(p[3])], device="cuda")
    s.ks = s.vs = s.mask = s.depth = None
    outlier = 1.0 + 3.0 * (torch.rand(G, 1, dim, generator=g, device="cuda") > 0.97)                       # some channels of keys are larger than others
    lay = (cap, n) if case["layout"] == "time" else (n, cap)
    k, v = rand(*lay, G, dim, dtype=F32).mul_(outlier.view(1, 1, G, dim)), rand(*lay, G, vdim, std=0.8, dtype=F32)
    if case["cache"] == "bf16":
        s.kc, s.vc = k.to(BF16), v.to(BF16)
    else:
        (s.kc, ks), (s.vc, vs) = _quantise(k, case["cache"], False), _quantise(v, case["cache"], False)
        s.ks, s.vs = ((x.permute(1, 2, 0) if case["layout"] == "time" else x.permute(0, 2, 1)).contiguous() for x in (ks, vs))
    if case["layout"] == "time":                                          # [positions, requests, heads, channels], seen request by request
        s.kc, s.vc = s.kc.permute(1, 0, 2, 3), s.vc.permute(1, 0, 2, 3)
    if case["branch"]:
        words, masks, depths = (s.rows + 63) // 64, [], []
        for _, _, _, m in portions:
            seen, deep = [], []
            for j, p in enumerate(_parents(case, m)):
                seen.append((seen[p] if p >= 0 else 0) | 1 << j)
                deep.append(deep[p] + 1 if p >= 0 else 0)
            masks += seen
            depths += deep
        signed = [[(w >> 64 * i & (1 << 64) - 1) - ((w >> 64 * i + 63 & 1) << 64) for i in range(words)] for w in masks]
        s.mask = torch.tensor(signed, dtype=torch.int64, device="cuda")
        s.depth = torch.tensor(depths, dtype=torch.int32, device="cuda")
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    if own:
        return _run_own(s)
    kind = s.case["kind"]
    if kind == "logprob":
        return _plain_logprob(s)
    if kind == "attn":
        return _plain_attn(s)
    if kind != "load":
        _plain_store(s)
    if kind == "store":
        return s.kc, s.ks, s.vc, s.vs
    s.k_out.copy_(_plain_load(s, s.kc, s.ks))
    s.v_out.copy_(_plain_load(s, s.vc, s.vs))
    return (s.k_out, s.v_out) if kind == "load" else (s.k_out, s.v_out, s.ks, s.vs)


def _run_own(s):
    from lia_b200 import ops
    c = s.case
    if c["kind"] == "logprob":
        return ops.token_logprobs(s.logits, s.tokens, top=c["top"])
    if c["kind"] == "attn":
        return ops.tree_attn(s.q, s.kc, s.vc, s.segs, s.out, c["H"], c["G"], c["dim"], c["vdim"], s.scale, rows=s.rows, max_ctx=s.max_ctx, mask=s.mask, depth=s.depth,
                             temp=s.temp, window=c["window"], softcap=c["softcap"], k_scale=s.ks, v_scale=s.vs)
    if c["kind"] != "load":
        ops.kv_store_8bit(s.k, s.v, s.meta, s.kc, s.vc, s.ks, s.vs, c["G"], c["dim"], c["vdim"], eps=EPS, norm_values=c["norm"])
    if c["kind"] == "store":
        return s.kc, s.ks, s.vc, s.vs
    ops.kv_load_8bit(s.meta, s.kc, s.vc, s.ks, s.vs, s.k_out, s.v_out, c["G"], c["dim"], c["vdim"])
    return (s.k_out, s.v_out) if c["kind"] == "load" else (s.k_out, s.v_out, s.ks, s.vs)


def _plain_put(s, x, d, norm, codes, scales):
    c, a = _quantise(x.float().view(s.M, -1, d), s.case["cache"], norm)
    codes.view(U8)[s.slot, s.pos] = c.view(U8).view(s.M, -1)
    scales[s.slot, :, s.pos] = a


def _plain_store(s):
    _plain_put(s, s.k, s.case["dim"], False, s.kc, s.ks)
    _plain_put(s, s.v, s.case["vdim"], s.case["norm"], s.vc, s.vs)


def _plain_load(s, codes, scales):
    x = codes.view(U8)[s.slot, s.pos].view(codes.dtype).float()
    return (x.view(s.M, s.case["G"], -1) * scales[s.slot, :, s.pos][..., None]).view(s.M, -1)


def _plain_rows(s, cache, scales, slots, T):
    """The first T positions of the portions' requests as numbers, [portions, heads, T, channels]."""
    c = s.case
    raw = cache.view(s.segs.shape[0], s.cap, c["G"], -1) if cache.dim() == 3 else cache
    x = (raw if raw.dtype == BF16 else raw.view(U8))[slots, :T].view(raw.dtype).float().permute(0, 2, 1, 3)
    return x if scales is None else x * scales[slots, :, :T][..., None]


def _plain_attn(s):
    c, dev = s.case, s.q.device
    H, G, dim, vdim, L, T = c["H"], c["G"], c["dim"], c["vdim"], s.rows, s.max_ctx
    slots, p0, row0, lens = s.segs.long().unbind(1)
    k, v = _plain_rows(s, s.kc, s.ks, slots, T), _plain_rows(s, s.vc, s.vs, slots, T)
    at = torch.arange(L, device=dev)
    rows = (row0[:, None] + at).clamp(max=s.M - 1)                                       # [portions, L]; rows behind a portion's end are dropped below
    q = s.q.float()[rows].view(-1, L, G, H // G, dim).permute(0, 2, 1, 3, 4).reshape(-1, G, L * (H // G), dim)
    x = (q @ k.transpose(2, 3) * s.scale).view(-1, G, L, H // G, T)
    if s.temp is not None:
        x = x * s.temp.view(G, 1, H // G, 1)
    if c["softcap"]:
        x = c["softcap"] * torch.tanh(x / c["softcap"])
    t = torch.arange(T, device=dev)
    behind = t[None, :] - p0[:, None]                                                    # < 0: history, else the number of a drafted token
    depth = at.expand(len(p0), L) if s.depth is None else s.depth.long()[rows]
    window = c["window"] if c["window"] else 1 << 40
    near = (depth[:, :, None] - behind[:, None, :]) < window
    if s.mask is None:
        sees = (behind[:, None, :] <= at[None, :, None]) & near
    else:
        j = behind.clamp(0, 64 * s.mask.shape[1] - 1)
        word = s.mask[rows].gather(2, (j >> 6)[:, None, :].expand(-1, L, -1))
        drafted = ((word >> (j & 63)[:, None, :]) & 1).bool() & (behind < lens[:, None])[:, None, :]
        sees = torch.where(behind[:, None, :] < 0, near, drafted)
    x = x.masked_fill(~sees[:, None, :, None, :], -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = (p.view(-1, G, L * (H // G), T) @ v).view(-1, G, L, H // G, vdim).permute(0, 2, 1, 3, 4).reshape(-1, L, H * vdim)
    s.out.copy_(o[s.row_seg, s.row_at])
    return s.out


def _plain_logprob(s):
    x = s.logits.float()
    e = x - x.amax(-1, keepdim=True)
    w = torch.exp(e)
    total = w.sum(-1, keepdim=True)
    logp = e - torch.log(total)
    entropy = -(w / total * logp.masked_fill(w == 0, 0.0)).sum(-1)
    ids = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, : s.case["top"]]         # of equal ones the lowest first
    return logp.gather(1, s.tokens), entropy, logp.gather(1, ids), ids


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["kind"] == "logprob":
        M, n = case["rows"], case["rows"] * case["vocab"]
        return {"bytes": n * (2 if case["act"] == "bf16" else 4) + M * (12 * case["given"] + 4 + 12 * case["top"]), "flops": 6 * n}
    portions = _portions(case)
    G, dim, vdim = case["G"], case["dim"], case["vdim"]
    if case["kind"] != "attn":
        M = portions[-1][2] + portions[-1][3]
        x, codes = M * G * (dim + vdim) * (2 if case["act"] == "bf16" else 4), M * G * (dim + vdim + 8) + 8 * M
        return {"bytes": x + codes if case["kind"] != "round" else 2 * (x + codes), "flops": 4 * M * G * (dim + vdim)}
    H, M, moved, pairs = case["H"], 0, 0, 0
    per_key = G * (2 * (dim + vdim) if case["cache"] == "bf16" else dim + vdim + 8)
    for _, past, _, m in portions:
        seen = min(past, case["window"] - 1) if case["window"] else past
        M += m
        moved += (seen + m) * per_key
        if case["branch"]:
            deep, own_keys = [], 0
            for p in _parents(case, m):
                deep.append(deep[p] + 1 if p >= 0 else 0)
                own_keys += deep[-1] + 1
            pairs += own_keys + m * seen
        else:
            far = case["window"] or 1 << 40
            pairs += sum(min(past + j + 1, far) for j in range(m))
    return {"bytes": moved + M * H * (dim + vdim) * 2 + (16 * M if case["branch"] else 0), "flops": 2 * (dim + vdim) * H * pairs}


# ------------------------------------------------------------------------------------------------ the same in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "logprob":
        return _exact_logprob(s)
    if case["kind"] == "attn":
        return _exact_attn(s)
    if case["kind"] == "load":
        return tuple(_exact_numbers(c, a, s) for c, a in ((s.kc, s.ks), (s.vc, s.vs)))
    got = []
    for x, d, norm in ((s.k, case["dim"], False), (s.v, case["vdim"], case["norm"])):
        x = x.double().view(s.M, case["G"], d)
        if norm:
            x = x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
        largest = x.abs().max(-1)[0].clamp(min=LEAST)
        if case["cache"] == "int8":
            step = largest / 127
            code = torch.round(x * 127 / largest[..., None])
        else:
            step = torch.exp2(torch.round(torch.log2(largest / 448)))
            step = torch.where(step * 448 < largest, 2 * step, torch.where(step * 224 >= largest, step / 2, step))
            y = x / step[..., None]
            grain = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)      # the distance of neighbouring codes
            code = torch.round(y / grain) * grain
        got.append((code, step))
    if case["kind"] == "round":
        return tuple((c * a[..., None]).reshape(s.M, -1) for c, a in got) + tuple(_placed(s, s.ks.shape, a.permute(0, 1), True) for _, a in got)
    return tuple(x for (c, a), codes in zip(got, (s.kc, s.vc)) for x in (_placed(s, codes.shape, c.reshape(s.M, -1), False), _placed(s, s.ks.shape, a, True)))


def _placed(s, shape, x, scales):
    out = torch.zeros(shape, dtype=F64, device="cuda")
    for i in range(shape[0]):
        mine = s.slot == i
        if scales:
            out[i][:, s.pos[mine]] = x[mine].t()
        else:
            out[i][s.pos[mine]] = x[mine]
    return out


def _exact_numbers(codes, scales, s):
    out = []
    for slot, first, _, m in _portions(s.case):
        c = codes[slot, first:first + m].double().view(m, s.case["G"], -1)
        out.append((c * scales[slot, :, first:first + m].double().t()[:, :, None]).reshape(m, -1))
    return torch.cat(out)


def _exact_attn(s):
    c = s.case
    H, G, dim, vdim = c["H"], c["G"], c["dim"], c["vdim"]
    if 4 * dim * H * sum((p[1] + p[3]) * p[3] for p in _portions(c)) > 2e11:
        return None
    out = torch.empty(s.M, H, vdim, dtype=F64, device="cuda")
    heads = [x.view(x.shape[0], x.shape[1], G, -1) if x.dim() == 3 else x for x in (s.kc, s.vc)]
    for slot, p0, row, m in _portions(c):
        T = p0 + m
        place = torch.arange(T, device="cuda")
        deep = s.depth[row:row + m].long() if s.depth is not None else torch.arange(m, device="cuda")
        sees = torch.ones(m, T, dtype=torch.bool, device="cuda")
        if c["branch"]:
            family = _parents(c, m)
            tree = torch.zeros(m, m, dtype=torch.bool)
            for j in range(m):
                a = j
                while a >= 0:
                    tree[j, a] = True
                    a = family[a]
            sees[:, p0:] = tree.to("cuda")
        else:
            sees[:, p0:] = torch.tril(sees[:, p0:])
        if c["window"]:
            far = place[None, :] <= (p0 + deep)[:, None] - c["window"]
            if c["branch"]:
                far[:, p0:] = False
            sees &= ~far
        for g in range(G):
            k, v = (x[slot, :T, g].double() for x in heads)
            if s.ks is not None:
                k, v = k * s.ks[slot, g, :T, None].double(), v * s.vs[slot, g, :T, None].double()
            for h in range(g * (H // G), (g + 1) * (H // G)):
                x = s.q[row:row + m, h * dim:(h + 1) * dim].double() @ k.t() * s.scale
                if s.temp is not None:
                    x = x * s.temp[h].double()
                if c["softcap"]:
                    x = torch.tanh(x / c["softcap"]) * c["softcap"]
                out[row:row + m, h] = torch.softmax(torch.where(sees, x, torch.full_like(x, -math.inf)), -1) @ v
    return out.view(s.M, H * vdim)


def _exact_logprob(s):
    M, top = s.case["rows"], s.case["top"]
    logp, entropy, best = [], [], []
    for r in range(0, M, 256):
        x = s.logits[r:r + 256].double()
        y = x - torch.logsumexp(x, -1, keepdim=True)
        logp.append(y.gather(1, s.tokens[r:r + 256]))
        entropy.append(-torch.special.xlogy(y.exp(), y.exp()).sum(-1))
        best.append(y.topk(top, -1)[0])
    return torch.cat(logp), torch.cat(entropy), torch.cat(best), None
