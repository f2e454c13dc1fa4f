"""The operators of serving in fewer bits, by which their speed is followed: keys and values stored in 4 bits and read back, attention over such caches,
projections in 8-bit integers, histories copied to other requests (forks) and drafted tokens moved to their places (compaction).

``prepare`` makes inputs, weights and caches on the GPU from the seed; ``run`` is one call of a user's program: of the package's operators, or, where
``own`` is false, of their plain form in elementary torch operations; ``exact`` is the same result in 64 bits.
"""
import math
import types

import torch

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
U8, I8 = torch.uint8, torch.int8
ACT = {"bf16": BF16, "f32": F32}
EPS = 1e-6
LEAST = 2.0 ** -100                 # a group's (a token's) largest number counts as at least that when its scale is chosen
GROUP = 32                          # channels that share a scale of a 4-bit cache

own = False


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # the keys and values of one decoded token of four requests into 4-bit caches and back, as a layer without a kernel for them would
        {"name": "round_token", "kind": "round", "act": "bf16", "seqs": 4, "tokens": 1, "past": 1900, "G": 8, "dim": 128, "vdim": 128, "norm": False},
        # four whole prompts of 2048 tokens, values normed per head on their way into the cache (Bebulorn)
        {"name": "round_prompts", "kind": "round", "act": "bf16", "seqs": 4, "tokens": 2048, "past": 0, "G": 8, "dim": 128, "vdim": 128, "norm": True},
        # trees of 29 drafted tokens behind histories of unequal odd lengths, under a sliding window with capped scores (Bebulorn's attention)
        {"name": "attn_tree_ragged", "kind": "attn", "seqs": 5, "past": 4099, "spread": 0.7, "tokens": 29, "branch": 2, "H": 16, "G": 8, "dim": 128, "vdim": 128, "window": 1024, "softcap": 50.0},
        # one decoded token of 16 requests with long histories: what 4 bits are for
        {"name": "attn_token_long", "kind": "attn", "seqs": 16, "past": 30001, "spread": 0.3, "tokens": 1, "branch": 0, "H": 16, "G": 8, "dim": 128, "vdim": 128, "window": 0, "softcap": 0.0},
        # the next portions of two prompts, of unequal odd lengths
        {"name": "attn_portions", "kind": "attn", "seqs": 2, "past": 512, "spread": 0.3, "tokens": 1003, "branch": 0, "H": 16, "G": 8, "dim": 128, "vdim": 128, "window": 0, "softcap": 0.0},
        # one token through a square projection of OPT-2.7b's width: latency
        {"name": "proj_token", "kind": "proj", "act": "bf16", "rows": 1, "K": 2560, "N": 2560},
        # the headline benchmark's decode step (batch 64) through the first projection of OPT-30B's feed-forward
        {"name": "proj_decode", "kind": "proj", "act": "bf16", "rows": 64, "K": 7168, "N": 28672},
        # a part of its prompts through the same: the largest
        {"name": "proj_prompt", "kind": "proj", "act": "bf16", "rows": 4096, "K": 7168, "N": 28672},
        # a prompt of 2049 tokens shared by 7 further answers: bf16 caches of 4 layers
        {"name": "fork_answers", "kind": "fork", "cache": "bf16", "layers": 4, "slots": 8, "sources": 1, "targets": 7, "count": 2049, "G": 8, "dim": 128},
        # two requests that branch into two, over 8-bit caches with their scales and a recurrent state a layer
        {"name": "fork_pairs", "kind": "fork", "cache": "int8", "layers": 6, "slots": 5, "sources": 2, "targets": 1, "count": 301, "G": 8, "dim": 128},
        # the accepted path of each of 16 drafted trees moves behind its history, bf16 caches of 12 layers
        {"name": "compact_trees", "kind": "compact", "cache": "bf16", "layers": 12, "seqs": 16, "past": 1901, "tokens": 29, "most": 6, "G": 8, "dim": 128},
        # the same of 64 requests over 4-bit caches of 15 layers
        {"name": "compact_batch", "kind": "compact", "cache": "int4", "layers": 15, "seqs": 64, "past": 280, "tokens": 64, "most": 9, "G": 8, "dim": 128},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(("round", "attn", "attn", "attn", "proj", "proj", "proj", "fork", "compact"))
    if kind == "proj":
        K, N = _log(rng, 64, 8192), _log(rng, 64, 30000)
        rows = _log(rng, 1, max(1, min(4096, 800_000_000_000 // (K * N))))
        return {"kind": kind, "act": rng.choice(("bf16", "bf16", "f32")), "rows": rows, "K": K, "N": N}
    dims = rng.choice(((128, 128), (128, 128), (64, 64), (64, 128), (128, 64)))
    if kind == "round":
        seqs, G = rng.randint(1, 16), rng.choice((1, 2, 3, 8, 12))
        return {"kind": kind, "act": rng.choice(("bf16", "bf16", "f32")), "seqs": seqs, "tokens": _log(rng, 1, 30000 // (seqs * G) + 1), "past": _log(rng, 1, 2000), "G": G,
                "dim": dims[0], "vdim": dims[1], "norm": rng.random() < 0.4}
    if kind == "fork":
        sources, targets = rng.randint(1, 3), rng.randint(1, 7)
        return {"kind": kind, "cache": rng.choice(("bf16", "int8", "int4")), "layers": rng.randint(1, 8), "slots": sources * (1 + targets) + rng.randint(0, 2), "sources": sources,
                "targets": targets, "count": _log(rng, 1, 1500), "G": rng.choice((1, 3, 8)), "dim": dims[0]}
    if kind == "compact":
        most = rng.randint(1, 12)
        return {"kind": kind, "cache": rng.choice(("bf16", "int8", "int4")), "layers": rng.randint(1, 15), "seqs": _log(rng, 1, 64), "past": _log(rng, 1, 2000),
                "tokens": rng.randint(2 * most, 64), "most": most, "G": rng.choice((1, 3, 8)), "dim": dims[0]}
    G, rep = rng.choice(((1, 8), (2, 4), (8, 1), (8, 2), (8, 4), (12, 1), (56, 1), (3, 5), (1, 1)))
    H, style = G * rep, rng.choice(("token", "token", "drafts", "drafts", "portions"))
    branch = rng.choice((0, 1, 2, 3)) if style != "portions" else 0
    seqs = _log(rng, 1, 64 if style != "portions" else 4)
    tokens = 1 if style == "token" else _log(rng, 2, 64) if style == "drafts" else _log(rng, 65, 1000)
    past = _log(rng, 1, min(60000, max(8, (1 << 26) // (seqs * max(G * 128, H * tokens // 2)))))
    return {"kind": kind, "seqs": seqs, "past": past, "spread": rng.choice((0.0, 0.5, 0.9)), "tokens": tokens, "branch": branch, "H": H, "G": G, "dim": dims[0], "vdim": dims[1],
            "window": rng.choice((0, 0, _log(rng, 64, 4096))), "softcap": rng.choice((0.0, 0.0, 30.0))}


# ------------------------------------------------------------------------------------------------ inputs
def _portions(case):
    """(slot, first position, first row, rows) of every request: slots in an order of their own, histories and portions a little shorter each time."""
    out, row, n = [], 0, case["seqs"]
    for i in range(n):
        past = int(case["past"] * (1 - case.get("spread", 0.0) * i / n))
        tokens = max(1, case["tokens"] - (case["tokens"] * i // (3 * n) if case["kind"] == "round" or case.get("spread") else 0))
        out.append((n - 1 - i, past, row, tokens))
        row += tokens
    return out


def _parents(case, n):
    return [(j - 1) // case["branch"] if j else -1 for j in range(n)]


def _quantise4(x):
    """x [.., dim] in 32 or 64 bits -> codes [.., dim] of -7 to 7, scales bf16 [.., dim / 32]: a / 7 of a group's largest magnitude a, in 32 bits and then rounded to 16."""
    y = x.view(*x.shape[:-1], -1, GROUP)
    a = y.abs().amax(-1)
    bad, a = ~torch.isfinite(a), a.clamp(min=LEAST)
    scale = (a / 7).float().to(BF16)
    codes = torch.round(y.double() / scale.double()[..., None]).masked_fill(bad[..., None], 0.0)      # (in 64 bits: next to a border 32 may choose the other code)
    return codes.view(x.shape), scale.masked_fill(bad, math.nan)


def _pack4(codes):
    """codes [.., dim] -> bytes [.., dim / 2]: code + 8 in 4 bits, the four channels 32 g + 4 q .. of a group g side by side (the lower channel in the lower bits), first by q, then by g"""
    u = (codes + 8).to(torch.int32).view(*codes.shape[:-1], -1, 8, 2, 2)
    return (u[..., 0] + 16 * u[..., 1]).transpose(-3, -2).reshape(*codes.shape[:-1], -1).to(U8)


def _unpack4(raw):
    """The reverse, in 32 bits"""
    b = raw.view(*raw.shape[:-1], 8, -1, 2).transpose(-3, -2)
    return torch.stack((b & 15, b >> 4), -1).reshape(*raw.shape[:-1], -1).float() - 8


def _numbers4(raw, scales):
    """bytes [.., dim / 2], scales [.., dim / 32] -> numbers"""
    c = _unpack4(raw)
    return (c.view(*c.shape[:-1], -1, GROUP) * scales.float()[..., None]).view(c.shape)


def _quantise8(x):
    """x [rows, K] -> int8 codes and a scale a row: the largest magnitude becomes 127"""
    a = x.abs().amax(-1, keepdim=True)
    bad, a = ~torch.isfinite(a), a.clamp(min=LEAST)
    codes = torch.round(127 * x / a).masked_fill(bad, 0.0)
    return codes, (a / 127).masked_fill(bad, math.nan)[:, 0]


def _caches(case, slots, cap, rand):
    """The caches of `layers` layers, keys and values, as a serving program keeps them: lists of (tensor, axis of positions)"""
    G, dim, out = case["G"], case["dim"], []
    for _ in range(2 * case["layers"]):
        if case["cache"] == "bf16":
            out.append((rand(slots, cap, G * dim), 1))
        else:
            out.append((torch.randint(0, 256, (slots, cap, G * dim // (2 if case["cache"] == "int4" else 1)), generator=rand.g, device="cuda", dtype=torch.int16).to(U8), 1))
            out.append((rand(slots, G, cap, dtype=F32), 2) if case["cache"] == "int8" else (rand(slots, G, cap, dim // GROUP), 2))
    return out


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 7013 + 29)

    def rand(*shape, std=1.0, mean=0.0, dtype=BF16):
        return (torch.randn(*shape, generator=g, device="cuda") * std + mean).to(BF16).to(dtype)

    rand.g = g
    s = types.SimpleNamespace(case=case, set=None)
    if case["kind"] == "proj":
        M, K, N = case["rows"], case["K"], case["N"]
        outlier = 1.0 + 9.0 * (torch.rand(K, generator=g, device="cuda") > 0.99)               # some channels of activations are larger than others
        s.x = (torch.randn(M, K, generator=g, device="cuda") * outlier).to(ACT[case["act"]])
        w = torch.randn(N, K, generator=g, device="cuda") * K ** -0.5
        codes, s.w_scale = _quantise8(w)
        s.w = torch.zeros(N, (K + 15) // 16 * 16, dtype=I8, device="cuda")[:, :K]               # rows are whole 16-byte vectors apart
        s.w.copy_(codes)
        s.out = torch.empty(M, N, dtype=ACT[case["act"]], device="cuda")
        return s
    if case["kind"] == "fork":
        n, per = case["sources"], case["targets"]
        cap = case["count"] + 7
        s.caches = _caches(case, case["slots"], cap, rand)
        s.states = [rand(case["slots"], 8, 64, 64, dtype=F32) for _ in range(case["layers"])] if case["cache"] == "int8" else []
        s.copies = [(i, n + i * per + j, max(1, case["count"] - 31 * i)) for i in range(n) for j in range(per)]      # (from, to, positions)
        s.on_gpu = torch.tensor(s.copies, dtype=torch.int32, device="cuda")
        return s
    if case["kind"] == "compact":
        n, T, most = case["seqs"], case["tokens"], case["most"]
        s.portions = [(n - 1 - i, case["past"] - case["past"] * i // (2 * n), i * T, T) for i in range(n)]
        s.caches = _caches(case, n, case["past"] + T + 3, rand)
        s.segs = torch.tensor(s.portions, dtype=torch.int32, device="cuda")
        later = torch.rand(n, T - most, generator=g, device="cuda").argsort(1)[:, : most - 1].sort(1)[0] + most     # a path: the root, then tokens behind the first `most`
        kept = torch.cat((torch.zeros(n, 1, dtype=torch.int64, device="cuda"), later), 1)
        length = 1 + torch.randint(0, most, (n, 1), generator=g, device="cuda")
        s.kept = kept.masked_fill(torch.arange(most, device="cuda") >= length, -1).to(torch.int32)
        s.kept_list = s.kept.tolist()
        return s
    portions = _portions(case)
    n, M = len(portions), portions[-1][2] + portions[-1][3]
    G, dim, vdim = case["G"], case["dim"], case["vdim"]
    cap = max(p[1] + p[3] for p in portions) + 5
    s.segs = torch.tensor(portions, dtype=torch.int32, device="cuda")
    s.M, s.cap, s.max_ctx, s.rows = M, cap, cap - 5, max(p[3] for p in portions)
    if case["kind"] == "round":
        s.meta = torch.tensor([(a, b + i) for a, b, _, m in portions for i in range(m)], dtype=torch.int32, device="cuda")
        s.k, s.v = rand(M, G * dim, std=1.5, dtype=ACT[case["act"]]), rand(M, G * vdim, std=0.7, dtype=ACT[case["act"]])
        s.slot, s.pos = s.meta[:, 0].long(), s.meta[:, 1].long()
        s.kc, s.vc = (torch.zeros(n, cap, G * d // 2, dtype=U8, device="cuda") for d in (dim, vdim))
        s.ks, s.vs = (torch.zeros(n, G, cap, d // GROUP, dtype=BF16, device="cuda") for d in (dim, vdim))
        s.k_out, s.v_out = torch.empty_like(s.k), torch.empty_like(s.v)
        return s
    H = case["H"]
    s.q = rand(M, H * dim, std=1.3)
    s.scale = dim ** -0.5
    s.temp = rand(H, std=0.1, mean=1.0, dtype=F32) if case["softcap"] else None
    s.out = torch.empty(M, H * vdim, dtype=BF16, device="cuda")
    s.row_seg = torch.tensor([i for i, p in enumerate(portions) for _ in range(p[3])], device="cuda")     # of every row: its portion, its place there
    s.row_at = torch.tensor([j for p in portions for j in range(p[3])], device="cuda")
    s.mask = s.depth = None
    outlier = 1.0 + 3.0 * (torch.rand(G, 1, dim, generator=g, device="cuda") > 0.97)                       # some channels of keys are larger than others
    for d, std, by, name in ((dim, 1.0, outlier, "k"), (vdim, 0.8, 1.0, "v")):
        raw = torch.empty(n, cap, G * d // 2, dtype=U8, device="cuda")
        scales = torch.empty(n, G, cap, d // GROUP, dtype=BF16, device="cuda")
        for i in range(n):                                                                                 # (request by request: a long history in 64 bits is large)
            c, a = _quantise4(rand(G, cap, d, std=std, dtype=F32) * by)
            raw[i].view(cap, G, d // 2).copy_(_pack4(c).transpose(0, 1))
            scales[i] = a
        setattr(s, name + "c", raw)
        setattr(s, name + "s", scales)
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
    kind = s.case["kind"]
    if own:
        return _run_own(s)
    if kind == "proj":
        return _plain_proj(s)
    if kind == "attn":
        return _plain_attn(s)
    if kind == "round":
        for x, d, norm, raw, scales, out in ((s.k, s.case["dim"], False, s.kc, s.ks, s.k_out), (s.v, s.case["vdim"], s.case["norm"], s.vc, s.vs, s.v_out)):
            _plain_put(s, x, d, norm, raw, scales)
            out.copy_(_numbers4(raw[s.slot, s.pos].view(s.M, s.case["G"], -1), scales[s.slot, :, s.pos]).view(s.M, -1))
        return s.k_out, s.v_out, s.ks, s.vs
    for t, axis in s.caches:
        x = t if axis == 1 else t.transpose(1, 2)
        if kind == "fork":
            for a, b, count in s.copies:
                x[b, :count] = x[a, :count]
        else:
            slot, p0, i = s.segs[:, :1].long(), s.segs[:, 1:2].long(), torch.arange(s.kept.shape[1], device=t.device)
            x[slot, p0 + i] = x[slot, p0 + torch.where(s.kept >= 0, s.kept, i)]      # (places behind a path's end keep what they hold)
    if kind == "fork":
        for t in s.states:
            for a, b, _ in s.copies:
                t[b] = t[a]
    return [t for t, _ in s.caches] + getattr(s, "states", [])


def _run_own(s):
    from lia_b200 import ops
    c = s.case
    if c["kind"] == "proj":
        return ops.linear_int8(s.x, s.w, s.w_scale, out=s.out)
    if c["kind"] == "attn":
        return ops.tree_attn(s.q, s.kc, s.vc, s.segs, s.out, c["H"], c["G"], c["dim"], c["vdim"], s.scale, rows=s.rows, max_ctx=s.max_ctx, mask=s.mask, depth=s.depth,
                             temp=s.temp, window=c["window"], softcap=c["softcap"], k_scale=s.ks, v_scale=s.vs)
    if c["kind"] == "round":
        ops.kv_store_4bit(s.k, s.v, s.meta, s.kc, s.vc, s.ks, s.vs, c["G"], c["dim"], c["vdim"], eps=EPS, norm_values=c["norm"])
        ops.kv_load_4bit(s.meta, s.kc, s.vc, s.ks, s.vs, s.k_out, s.v_out, c["G"], c["dim"], c["vdim"])
        return s.k_out, s.v_out, s.ks, s.vs
    if s.set is None:                                                                # a handle of the caches, which a serving program makes with them
        s.set = ops.CacheSet([t if axis == 1 else t.transpose(1, 2) for t, axis in s.caches], getattr(s, "states", []))
    if c["kind"] == "fork":
        s.set.fork(s.on_gpu, max_count=c["count"])
    else:
        s.set.compact(s.segs, s.kept)
    return [t for t, _ in s.caches] + getattr(s, "states", [])


def _plain_put(s, x, d, norm, raw, scales):
    x = x.float().view(s.M, -1, d)
    if norm:
        x = (x.double() / torch.sqrt(x.double().square().mean(-1, keepdim=True) + EPS)).float()      # (in 64 bits and rounded once: what lies next to a border counts)
    c, a = _quantise4(x)
    raw[s.slot, s.pos] = _pack4(c).view(s.M, -1)
    scales[s.slot, :, s.pos] = a


def _plain_proj(s):
    codes, scale = _quantise8(s.x.float())
    sums = torch.cat([codes.double() @ s.w[i:i + 8192].double().t() for i in range(0, s.w.shape[0], 8192)], 1)    # (whole numbers beyond 2^24: in 64 bits)
    s.out.copy_(sums.float() * scale[:, None] * s.w_scale)
    return s.out


def _plain_attn(s):
    c, dev = s.case, s.q.device
    H, G, dim, vdim, L, T = c["H"], c["G"], c["dim"], c["vdim"], s.rows, s.max_ctx
    slots, p0, row0, lens = s.segs.long().unbind(1)
    n = len(slots)
    k, v = (_numbers4(raw[slots, :T].view(n, T, G, -1).transpose(1, 2), a[slots, :, :T]) for raw, a in ((s.kc, s.ks), (s.vc, s.vs)))
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
    depth = at.expand(n, L) if s.depth is None else s.depth.long()[rows]
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


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def _position_bytes(case):
    """of one position of all the caches of a fork or a compaction"""
    per = {"bf16": 2 * case["dim"], "int8": case["dim"] + 4, "int4": case["dim"] // 2 + case["dim"] // 16}[case["cache"]]
    return 2 * case["layers"] * case["G"] * per


def work(case):
    if case["kind"] == "proj":
        M, K, N = case["rows"], case["K"], case["N"]
        act = 2 if case["act"] == "bf16" else 4
        return {"bytes": N * (K + 4) + M * (K + N) * act, "flops": 2 * M * N * K}
    if case["kind"] == "fork":
        state = 4 * 8 * 64 * 64 * case["layers"] if case["cache"] == "int8" else 0
        moved = sum(max(1, case["count"] - 31 * i) * _position_bytes(case) + state for i in range(case["sources"]))
        return {"bytes": moved * (1 + case["targets"]), "flops": 0}
    if case["kind"] == "compact":                                                        # on average half of a path is there, of which the root stays where it is
        return {"bytes": int(2 * case["seqs"] * (case["most"] - 1) / 2 * _position_bytes(case)) + 1, "flops": 0}
    portions = _portions(case)
    G, dim, vdim = case["G"], case["dim"], case["vdim"]
    per_key = G * ((dim + vdim) // 2 + (dim + vdim) // 16)
    if case["kind"] == "round":
        M = portions[-1][2] + portions[-1][3]
        x = M * G * (dim + vdim) * (2 if case["act"] == "bf16" else 4)
        return {"bytes": 2 * (x + M * per_key + 8 * M), "flops": 4 * M * G * (dim + vdim)}
    H, M, moved, pairs = case["H"], 0, 0, 0
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
    if case["kind"] == "proj":
        x = s.x.double()
        largest = x.abs().max(-1)[0].clamp(min=LEAST)
        codes = torch.round(x * 127 / largest[:, None])
        return (codes @ s.w.double().t()) * (largest / 127)[:, None] * s.w_scale.double()
    if case["kind"] in ("fork", "compact"):
        return _exact_moved(s)
    if case["kind"] == "attn":
        return _exact_attn(s)
    numbers, scales = [], []
    for x, d, norm, like in ((s.k, case["dim"], False, s.ks), (s.v, case["vdim"], case["norm"], s.vs)):
        x = x.double().view(s.M, case["G"], d)
        if norm:
            x = x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
        y = x.unflatten(-1, (d // GROUP, GROUP))
        step = (y.abs().max(-1)[0].clamp(min=LEAST) / 7).to(F32).to(BF16).double()        # (a scale is what its 16 bits stand for)
        numbers.append((torch.round(y / step[..., None]) * step[..., None]).reshape(s.M, -1))
        placed = torch.zeros(like.shape, dtype=F64, device="cuda")
        for i in range(like.shape[0]):
            placed[i][:, s.pos[s.slot == i]] = step[s.slot == i].transpose(0, 1)
        scales.append(placed)
    return tuple(numbers + scales)


def _exact_moved(s):
    out = []
    for t, axis in s.caches:
        x = t.movedim(axis, 1)
        index = torch.arange(x.shape[0] * x.shape[1], device="cuda").view(x.shape[0], x.shape[1])    # of every place: where its content comes from
        if s.case["kind"] == "fork":
            for a, b, count in s.copies:
                index[b, :count] = a * x.shape[1] + torch.arange(count, device="cuda")
        else:
            for (slot, p0, _, _), kept in zip(s.portions, s.kept_list):
                for i, j in enumerate(kept):
                    if j >= 0:
                        index[slot, p0 + i] = slot * x.shape[1] + p0 + j
        out.append(x.reshape(-1, *x.shape[2:])[index].movedim(1, axis))
    for t in getattr(s, "states", []):
        came = list(range(t.shape[0]))
        for a, b, _ in s.copies:
            came[b] = a
        out.append(t[came])
    return out


def _exact_attn(s):
    c = s.case
    H, G, dim, vdim = c["H"], c["G"], c["dim"], c["vdim"]
    if 4 * dim * H * sum((p[1] + p[3]) * p[3] for p in _portions(c)) > 2e11:
        return None
    out = torch.empty(s.M, H, vdim, dtype=F64, device="cuda")

    def numbers(raw, scales, slot, g, T, d):
        b = raw[slot, :T].view(T, G, d // 2)[:, g].to(torch.int64)
        x = torch.empty(T, d, dtype=F64, device="cuda")
        channel = torch.arange(d, device="cuda")
        byte = 2 * (channel % GROUP // 4 * (d // GROUP) + channel // GROUP) + channel % 4 // 2
        x[:] = ((b[:, byte] >> (4 * (channel % 2))) % 16 - 8).double()
        return x * scales[slot, g, :T].double().repeat_interleave(GROUP, 1)

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
            k, v = numbers(s.kc, s.ks, slot, g, T, dim), numbers(s.vc, s.vs, slot, g, T, vdim)
            for h in range(g * (H // G), (g + 1) * (H // G)):
                x = s.q[row:row + m, h * dim:(h + 1) * dim].double() @ k.t() * s.scale
                if s.temp is not None:
                    x = x * s.temp[h].double()
                if c["softcap"]:
                    x = torch.tanh(x / c["softcap"]) * c["softcap"]
                out[row:row + m, h] = torch.softmax(torch.where(sees, x, torch.full_like(x, -math.inf)), -1) @ v
    return out.view(s.M, H * vdim)
