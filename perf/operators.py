"""Operators on long key/value caches, as cases that can be timed and compared.

Four operators share one cache (``capi.KVCache``):

* ``attend``     -- ``ncmb_cache_attention``: the new tokens of every row -- one, a run, or a tree of drafted ones -- attend to
  the row's cache and to their own ancestors; optionally every cached token's share of that attention is added up;
* ``evict``      -- ``ncmb_cache_evict``: each row and head of a cache is held to a budget of tokens by those added-up shares;
* ``summaries``  -- ``ncmb_block_summaries``: an 8-bit mean key for every block of cached tokens;
* ``blocks``     -- ``ncmb_block_attention``: every query picks blocks of the cache by those means and attends to them alone.

Shapes of heads are this repository's decoder and generator configurations (12 x 64, 14 over 2 x 64, 16 over 4 x 64) and the
generic 32 over 8 x 128. Caches are laid out token by token with keys and values side by side, as the library's own decode
loops hold them, or head by head.
"""
import functools
import math

import torch

own = False

HEADS = {"gpt2": (12, 12, 64), "qwen": (14, 2, 64), "box": (16, 4, 64), "wide": (32, 8, 128)}    # query heads, kv heads, head dim


# ------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # one interactive completion of the GPT-2 shape near the end of its context, fp32 cache: the smallest call, all latency
        {"name": "attend_gpt2_1x811", "op": "attend", "heads": "gpt2", "cache": "f32", "act": "f32", "layout": "token", "B": 1, "T": 1,
         "len": 811, "ragged": False, "tree": False, "weights": False},
        # one interactive user of the Qwen2 shape, a drafted tree of 23 tokens to verify
        {"name": "tree_qwen_1x4071", "op": "attend", "heads": "qwen", "cache": "bf16", "act": "f32", "layout": "token", "B": 1, "T": 23,
         "len": 4071, "ragged": False, "tree": True, "weights": False},
        # a server's batch with trees of up to 16 drafted tokens, rows of all lengths, one of them new
        {"name": "tree_wide_16x8192", "op": "attend", "heads": "wide", "cache": "bf16", "act": "bf16", "layout": "head", "B": 16, "T": 16,
         "len": 8192, "ragged": True, "tree": True, "weights": False},
        # a decode step of many rows that adds up the weights by which the cache will be trimmed
        {"name": "attend_qwen_64x16000_w", "op": "attend", "heads": "qwen", "cache": "bf16", "act": "f32", "layout": "token", "B": 64, "T": 1,
         "len": 16000, "ragged": True, "tree": False, "weights": True},
        # the last 32 tokens of prompts look back over them, to find out what to keep; fp32 cache
        {"name": "window_box_4x8000_w", "op": "attend", "heads": "box", "cache": "f32", "act": "f32", "layout": "token", "B": 4, "T": 32,
         "len": 8000, "ragged": False, "tree": False, "weights": True},
        # prompts of all lengths into small caches of their own
        {"name": "evict_prompt_16x8192", "op": "evict", "heads": "wide", "cache": "bf16", "layout": "head", "B": 16, "len": 8192,
         "budget": 1024, "recent": 128, "ragged": True, "inplace": False},
        # after each decode step: one token over budget
        {"name": "evict_step_64x2049", "op": "evict", "heads": "qwen", "cache": "bf16", "layout": "token", "B": 64, "len": 2049,
         "budget": 2048, "recent": 64, "ragged": False, "inplace": True},
        # means of a prompt's blocks, a few long rows
        {"name": "summaries_wide_4x32768", "op": "summaries", "heads": "wide", "cache": "bf16", "layout": "head", "B": 4, "len": 32768,
         "new": 32768, "block": 64, "ragged": False},
        # means of what a piece of a prompt appended, fp32 cache, odd lengths
        {"name": "summaries_box_16x5003", "op": "summaries", "heads": "box", "cache": "f32", "layout": "token", "B": 16, "len": 5003,
         "new": 1001, "block": 32, "ragged": True},
        # one user at 128K tokens
        {"name": "blocks_qwen_1x131000", "op": "blocks", "heads": "qwen", "cache": "bf16", "act": "f32", "layout": "token", "B": 1, "T": 1,
         "len": 131000, "block": 64, "n_sel": 32, "ragged": False},
        # a server's step over long rows of all lengths
        {"name": "blocks_wide_32x32768", "op": "blocks", "heads": "wide", "cache": "bf16", "act": "bf16", "layout": "head", "B": 32, "T": 1,
         "len": 32768, "block": 64, "n_sel": 32, "ragged": True},
        # a short run of tokens each with blocks of its own, fp32 cache
        {"name": "blocks_box_3x16001_t24", "op": "blocks", "heads": "box", "cache": "f32", "act": "f32", "layout": "token", "B": 3, "T": 24,
         "len": 16001, "block": 32, "n_sel": 48, "ragged": False},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


MOST_CACHE = 1 << 31      # bytes a drawn case's cache may take
MOST_WORK = 2.0e9         # and the plain form's largest intermediate, in elements


def draw(rng):
    while True:
        c = {"op": rng.choice(["attend", "attend", "evict", "summaries", "blocks", "blocks"]), "heads": rng.choice(list(HEADS)),
             "cache": rng.choice(["f32", "bf16", "bf16"]), "layout": rng.choice(["token", "head"]), "B": _log(rng, 1, 64),
             "len": _log(rng, 1, 40000), "ragged": rng.random() < 0.6}
        H, nkv, hd = HEADS[c["heads"]]
        es = 4 if c["cache"] == "f32" else 2
        if c["op"] in ("attend", "blocks"):
            c["act"] = "f32" if c["cache"] == "f32" else rng.choice(["f32", "bf16"])
            c["T"] = rng.choice([1, 1, _log(rng, 2, 64)])
        if c["op"] == "attend":
            c["tree"] = c["T"] > 1 and rng.random() < 0.6
            c["weights"] = rng.random() < 0.4
            big = c["B"] * c["T"] * H * c["len"]
        elif c["op"] == "evict":
            c["budget"] = _log(rng, 1, max(2, c["len"]))
            c["recent"] = rng.randint(0, c["budget"])
            c["inplace"] = c["len"] <= c["budget"] + 64
            big = c["B"] * nkv * c["len"] * hd
        elif c["op"] == "summaries":
            c["block"] = rng.choice([16, 32, 64, 128])
            c["new"] = _log(rng, 1, c["len"])
            big = c["B"] * nkv * c["len"] * hd
        else:
            c["block"] = rng.choice([16, 32, 64, 128])
            c["n_sel"] = rng.randint(3, 64)
            big = c["B"] * c["T"] * nkv * c["n_sel"] * c["block"] * hd * 2
        if big <= MOST_WORK / 4 and 2 * c["B"] * nkv * c["len"] * hd * es <= MOST_CACHE:
            return c


# ------------------------------------------------------------------------------------------- inputs

def _lens(case):
    """Tokens of each row: the stated length, or lengths from nothing up to it."""
    B, n = case["B"], case["len"]
    if not case["ragged"] or B == 1:
        return [n] * B
    out = [max(1, n * (16 + (b * 37 + 11) % 48) // 63) for b in range(B)]
    out[0] = n
    if case["op"] in ("attend", "summaries", "blocks"):
        out[1] = 0                                  # a row that has just been opened
    return [min(n, v) for v in out]


def _cache(case, cap, g):
    H, nkv, hd = HEADS[case["heads"]]
    dt = torch.float32 if case["cache"] == "f32" else torch.bfloat16
    B = case["B"]
    if case["layout"] == "token":                   # [row][token][keys | values of all heads]
        buf = torch.randn(B, cap, 2, nkv, hd, device="cuda", dtype=dt, generator=g)
        k, v = buf[:, :, 0].permute(0, 2, 1, 3), buf[:, :, 1].permute(0, 2, 1, 3)
    else:                                           # [row][head][token]
        k = torch.randn(B, nkv, cap, hd, device="cuda", dtype=dt, generator=g)
        v = torch.randn(B, nkv, cap, hd, device="cuda", dtype=dt, generator=g)
    if case["op"] in ("summaries", "blocks"):       # neighbouring tokens share a part of their keys
        run = 48
        part = torch.randn(B, nkv, cap // run + 1, hd, device="cuda", dtype=dt, generator=g)
        for i in range(cap // run + 1):
            k[:, :, i * run:(i + 1) * run] += part[:, :, i:i + 1]
    return k, v


def _parents(case, seed):
    """Random trees: a row's first nodes are roots or hang on one of the eight before; what is left of the row is unused."""
    import random
    r = random.Random(seed * 7919 + 5)
    rows = []
    for b in range(case["B"]):
        n = r.randint(max(1, case["T"] // 2), case["T"])
        rows.append([(-1 if t == 0 or r.random() < 0.05 else r.randint(max(0, t - 8), t - 1)) if t < n else -2 for t in range(case["T"])])
    return rows


def prepare(case, seed):
    H, nkv, hd = HEADS[case["heads"]]
    g = torch.Generator(device="cuda").manual_seed(int(seed) & 0x7fffffff)
    B, op = case["B"], case["op"]
    lens = _lens(case)
    T = case.get("T", 0)
    cap = case["len"] + T + 5
    s = {"case": case, "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"), "cap": cap, "max_len": max(lens)}
    s["k"], s["v"] = _cache(case, cap, g)
    if "act" in case:
        dt = torch.float32 if case["act"] == "f32" else torch.bfloat16
        s["q"] = torch.randn(B, T, H, hd, device="cuda", generator=g).mul_(1.5).to(dt)
        s["out"] = torch.empty(B, T, H, hd, device="cuda", dtype=dt)
    if op == "attend":
        s["parents"] = torch.tensor(_parents(case, int(seed)), dtype=torch.int32, device="cuda") if case["tree"] else None
        # what a handful of steps before this one has added up
        s["weights"] = torch.rand(B, nkv, cap, device="cuda", generator=g).mul_(8 * H / nkv / case["len"]) if case["weights"] else None
    elif op == "evict":
        # shares as attention gives them: a few large, most small, some tokens that nothing has looked at
        w = torch.randn(B, nkv, cap, device="cuda", generator=g).mul_(2).exp_()
        s["weights"] = w.masked_fill_(torch.rand(B, nkv, cap, device="cuda", generator=g) < 0.04, 0.0)
        known = min(case["budget"], case["len"] - 1) if case["inplace"] else 0
        s["known"] = torch.tensor([min(known, n) for n in lens], dtype=torch.int32, device="cuda")
        far = 3 * case["len"] if case["inplace"] else 0
        s["seen"] = torch.tensor([n + far for n in lens], dtype=torch.int32, device="cuda")
        # where the tokens that are known stood in their text: distinct places, in the order that earlier evictions left
        old = torch.rand(B, nkv, far + 1, device="cuda", generator=g).argsort(-1)[:, :, :known] if known else torch.zeros(B, nkv, 0, device="cuda")
        s["pos"] = torch.zeros(B, nkv, cap, dtype=torch.int32, device="cuda")
        s["pos"][:, :, :old.shape[2]] = old
        room = cap if case["inplace"] else min(case["budget"], case["len"])
        s["room"] = room
        if case["inplace"]:
            s["k2"], s["v2"], s["weights2"], s["pos2"] = s["k"], s["v"], s["weights"], s["pos"]
        else:
            s["k2"] = torch.zeros(B, nkv, room, hd, device="cuda", dtype=s["k"].dtype)
            s["v2"] = torch.zeros_like(s["k2"])
            s["weights2"] = torch.zeros(B, nkv, room, device="cuda")
            s["pos2"] = torch.zeros(B, nkv, room, dtype=torch.int32, device="cuda")
        s["lens2"] = torch.zeros(B, dtype=torch.int32, device="cuda")
    else:
        nb = -(-cap // case["block"])
        s["codes"] = torch.zeros(B, nkv, nb, hd, dtype=torch.int8, device="cuda")
        s["scales"] = torch.zeros(B, nkv, nb, device="cuda")
        if op == "summaries":
            s["first"] = torch.tensor([max(0, n - case["new"]) for n in lens], dtype=torch.int32, device="cuda")
        else:                                       # what ncmb_block_summaries has made of the cache by then
            for b in range(B):
                _summarise(s["k"][b:b + 1], case["block"], torch.zeros_like(s["lens"][b:b + 1]), s["lens"][b:b + 1] + T, s["codes"][b:b + 1], s["scales"][b:b + 1])
            s["picks"] = torch.empty(B, T, nkv, case["n_sel"], dtype=torch.int32, device="cuda")
    return s


# ------------------------------------------------------------------------------------------- plain forms

def _seen(lens, T, cap, parents):
    """[B][T][cap]: which slots a node sees -- its row's cached tokens, itself and its ancestors; [B][T]: nodes that are used."""
    B = lens.shape[0]
    t = torch.arange(T, device=lens.device)
    if parents is None:
        anc = (t[:, None] >= t[None, :]).expand(B, T, T)
        used = torch.ones(B, T, dtype=torch.bool, device=lens.device)
    else:
        p = parents.long()
        used = (p >= -1) & (p < t)
        link = (p[:, :, None] == t) & used[:, :, None]
        up = torch.eye(T, device=lens.device).expand(B, T, T) + link.float()
        for _ in range(max(1, (T - 1).bit_length())):        # paths of 1, 2, 4, ... steps
            up = (up @ up).clamp_(max=1.0)
        anc = (up > 0) & used[:, :, None] & used[:, None, :]
    at = torch.arange(cap, device=lens.device)[None, :] - lens.long()[:, None]        # [B][cap]: slot as a node's number
    own_ = anc.gather(2, at.clamp(0, T - 1)[:, None, :].expand(B, T, cap)) & ((at >= 0) & (at < T))[:, None, :]
    return (own_ | (at < 0)[:, None, :]) & used[:, :, None], used


def _softmax(s, seen):
    """Over the last axis, over what is seen; rows that see nothing are zero."""
    s = s.masked_fill(~seen, float("-inf"))
    m = s.amax(-1, keepdim=True)
    e = torch.exp(s - m.masked_fill(m == float("-inf"), 0.0))
    return e / e.sum(-1, keepdim=True).clamp_(min=1e-30)


def _attend(s):
    case = s["case"]
    H, nkv, hd = HEADS[case["heads"]]
    B, T, G, cap = case["B"], case["T"], H // nkv, s["cap"]
    q = s["q"].float().view(B, T, nkv, G, hd).permute(0, 2, 1, 3, 4).reshape(B, nkv, T * G, hd)
    k, v = s["k"].float(), s["v"].float()
    seen, _ = _seen(s["lens"], T, cap, s["parents"])
    sc = (q @ k.transpose(2, 3)).view(B, nkv, T, G, cap) * (1.0 / math.sqrt(hd))
    p = _softmax(sc, seen[:, None, :, None, :])
    out = (p.view(B, nkv, T * G, cap) @ v).view(B, nkv, T, G, hd).permute(0, 2, 1, 3, 4).reshape(B, T, H, hd).to(s["q"].dtype)
    if s["weights"] is None:
        return {"out": out}
    at = torch.arange(cap, device=out.device)[None, :] - s["lens"].long()[:, None]
    w = p.sum((2, 3))
    old = s["weights"]
    s["weights"].copy_(torch.where((at < 0)[:, None], old + w, torch.where((at < T)[:, None], w, old)))
    return {"out": out, "weights": s["weights"]}


def _evict(s):
    case = s["case"]
    B, room = case["B"], s["room"]
    nkv, cap = s["weights"].shape[1:]
    slot = torch.arange(cap, device="cuda")
    n, known, seen = (s[x].long()[:, None, None] for x in ("lens", "known", "seen"))
    live = (slot < n).expand(B, nkv, cap)
    pos = torch.where(slot < known, s["pos"].long(), seen - n + slot)
    last = pos.masked_fill(~live, -1).amax(-1, keepdim=True)
    keep_first = live & (pos > last - case["recent"])
    key = s["weights"].masked_fill(keep_first, float("inf")).masked_fill(~live, float("-inf"))
    order = key.sort(dim=-1, descending=True, stable=True).indices          # ties: the lower slot first
    n2 = n.clamp(max=case["budget"])
    rank = torch.empty_like(order).scatter_(-1, order, slot.expand(B, nkv, cap))
    kept = live & (rank < n2)
    stays = kept & (slot < n2)
    holes, movers = (slot < n2) & ~kept, kept & (slot >= n2)
    # the i-th freed slot takes the i-th kept token from beyond
    src = slot.expand(B, nkv, cap).clone()
    mover_at = (~movers).long().sort(dim=-1, stable=True).indices           # movers' slots first, ascending
    src = torch.where(holes, mover_at.gather(-1, (holes.long().cumsum(-1) - 1).clamp(min=0)), src)[:, :, :min(room, cap)]
    write = (slot < n2).expand(B, nkv, cap)[:, :, :src.shape[2]]
    if case["inplace"]:                                                 # what stays is not touched
        write = write & ~stays[:, :, :src.shape[2]]
    for x in ("k", "v"):
        s[x + "2"][:, :, :src.shape[2]] = torch.where(write[..., None], s[x].gather(2, src[..., None].expand(*src.shape, s[x].shape[3])), s[x + "2"][:, :, :src.shape[2]])
    new_w, new_pos = s["weights"].gather(2, src), pos.gather(2, src).int()
    inside = (slot < n2).expand(B, nkv, cap)[:, :, :src.shape[2]]
    s["weights2"][:, :, :src.shape[2]] = torch.where(inside, new_w, s["weights2"][:, :, :src.shape[2]])
    s["pos2"][:, :, :src.shape[2]] = torch.where(inside, new_pos, s["pos2"][:, :, :src.shape[2]])
    s["lens2"].copy_(n2.view(B))
    return {"k": s["k2"], "v": s["v2"], "weights": s["weights2"], "pos": s["pos2"], "len": s["lens2"]}


def _summarise(k, block, first, total, codes, scales):
    """Mean key of every block that holds a token of [first, total), in 8 bits. Sums run by halves of the block: token i and
    token i + n/2 are added, then the same of what is left."""
    B, nkv, cap, hd = k.shape
    nb = codes.shape[2]
    slot = torch.arange(nb * block, device=k.device)
    x = torch.zeros(B, nkv, nb * block, hd, device=k.device)
    x[:, :, :cap] = k.float()
    x.masked_fill_((slot >= total.long()[:, None])[:, None, :, None], 0.0)
    x = x.view(B, nkv, nb, block, hd)
    n = block
    while n > 1:
        n //= 2
        x = x[:, :, :, :n] + x[:, :, :, n:2 * n]
    at = torch.arange(nb, device=k.device)
    count = (total.long()[:, None] - at * block).clamp(1, block)
    mean = x[:, :, :, 0] / count[:, None, :, None].float()
    scale = mean.abs().amax(-1) / torch.full((), 127.0, device=k.device)
    code = torch.where(scale[..., None] > 0, torch.round(mean / scale[..., None]), torch.zeros_like(mean)).to(torch.int8)
    touched = ((at * block < total.long()[:, None]) & ((at + 1) * block > first.long()[:, None]))[:, None]
    codes.copy_(torch.where(touched[..., None], code, codes))
    scales.copy_(torch.where(touched, scale, scales))


def _summaries(s):
    _summarise(s["k"], s["case"]["block"], s["first"], s["lens"], s["codes"], s["scales"])
    return s["codes"] * s["scales"].unsqueeze(-1)


N_FIRST, N_LAST = 1, 2


def _pick(s):
    """[B][T][kv heads][n_sel] blocks in ascending order, -1 where there are fewer."""
    case = s["case"]
    H, nkv, hd = HEADS[case["heads"]]
    B, T, G, block, n_sel = case["B"], case["T"], H // nkv, case["block"], case["n_sel"]
    nb = s["codes"].shape[2]
    q = s["q"].float().view(B, T, nkv, G, hd)
    qs = q.abs().amax(-1, keepdim=True) / torch.full((), 127.0, device=q.device)
    q8 = torch.where(qs > 0, torch.round(q / qs), torch.zeros_like(q))
    dots = q8.permute(0, 2, 1, 3, 4).reshape(B, nkv, T * G, hd) @ s["codes"].float().transpose(2, 3)       # whole numbers
    dots = dots.view(B, nkv, T, G, nb) * qs.permute(0, 2, 1, 3, 4)
    score = (dots.amax(3) * s["scales"][:, :, None]).permute(0, 2, 1, 3)                      # [B][T][nkv][nb]
    cur = ((s["lens"].long()[:, None] + torch.arange(T, device=q.device)) // block)[:, :, None, None]
    at = torch.arange(nb, device=q.device)
    score = score.masked_fill((at < N_FIRST) | (at > cur - N_LAST), float("inf")).masked_fill(at > cur, float("-inf"))
    top = score.sort(dim=-1, descending=True, stable=True).indices[..., :n_sel]
    top = torch.nn.functional.pad(top, (0, max(0, n_sel - nb)), value=nb)
    top = torch.where((torch.arange(n_sel, device=q.device) <= cur) & (top <= cur), top, torch.full_like(top, nb)).sort(-1).values
    return torch.where(top < nb, top, torch.full_like(top, -1)).int()


def _blocks(s):
    case = s["case"]
    H, nkv, hd = HEADS[case["heads"]]
    B, T, G, block, n_sel, cap = case["B"], case["T"], H // nkv, case["block"], case["n_sel"], s["cap"]
    picks = _pick(s)
    p = picks.permute(0, 2, 1, 3).long()                                                      # [B][nkv][T][n_sel]
    tok = (p[..., None] * block + torch.arange(block, device=p.device)).view(B, nkv, T, n_sel * block)
    here = (s["lens"].long()[:, None] + torch.arange(T, device=p.device))[:, None, :, None]
    seen = (p >= 0).repeat_interleave(block, -1) & (tok <= here)
    tok = tok.clamp(0, cap - 1)
    b, h = torch.arange(B, device=p.device)[:, None, None, None], torch.arange(nkv, device=p.device)[None, :, None, None]
    k, v = s["k"][b, h, tok].float(), s["v"][b, h, tok].float()                               # [B][nkv][T][keys][hd]
    q = s["q"].float().view(B, T, nkv, G, hd).permute(0, 2, 1, 3, 4)
    w = _softmax((q @ k.transpose(3, 4)) * (1.0 / math.sqrt(hd)), seen[:, :, :, None])
    out = (w @ v).permute(0, 2, 1, 3, 4).reshape(B, T, H, hd).to(s["q"].dtype)
    return {"out": out, "picks": picks}


# ------------------------------------------------------------------------------------------- the framework's

@functools.lru_cache(maxsize=1)
def _library():
    import __graft_entry__
    pkg = __graft_entry__.load_package()
    return pkg.load_library(), pkg.capi


def _handle(s, k, v, n):
    """The library's view of a cache, which a program makes when it allocates one."""
    name = "handle_" + k
    if name not in s:
        s[name] = _library()[1].KVCache.of(s[k], s[v], s[n])
    return s[name]


def _ptr(t):
    return None if t is None else t.data_ptr()


def _run_own(s):
    lib, capi = _library()
    case = s["case"]
    H, nkv, hd = HEADS[case["heads"]]
    cache, op = _handle(s, "k", "v", "lens"), case["op"]
    if op in ("attend", "blocks"):
        act = capi.BF16 if case["act"] == "bf16" else capi.F32
    if op == "attend":
        rc = lib.ncmb_cache_attention(cache, s["q"].data_ptr(), H * hd, s["out"].data_ptr(), H * hd, act, H, case["T"], _ptr(s["parents"]), 0.0,
                                      s["max_len"], _ptr(s["weights"]))
        out = {"out": s["out"]} if s["weights"] is None else {"out": s["out"], "weights": s["weights"]}
    elif op == "evict":
        to = cache if case["inplace"] else _handle(s, "k2", "v2", "lens2")
        rc = lib.ncmb_cache_evict(cache, to, s["weights"].data_ptr(), s["weights2"].data_ptr(), s["pos"].data_ptr(), s["pos2"].data_ptr(),
                                  s["known"].data_ptr(), s["seen"].data_ptr(), case["budget"], case["recent"], s["max_len"], s["lens2"].data_ptr())
        out = {"k": s["k2"], "v": s["v2"], "weights": s["weights2"], "pos": s["pos2"], "len": s["lens2"]}
    elif op == "summaries":
        rc = lib.ncmb_block_summaries(cache, 0, s["first"].data_ptr(), case["block"], s["max_len"], s["codes"].data_ptr(), s["scales"].data_ptr())
        out = s["codes"] * s["scales"].unsqueeze(-1)
    else:
        rc = lib.ncmb_block_attention(cache, s["q"].data_ptr(), H * hd, s["out"].data_ptr(), H * hd, act, H, case["T"], case["block"],
                                      s["codes"].data_ptr(), s["scales"].data_ptr(), case["n_sel"], N_FIRST, N_LAST, 0.0, s["max_len"], s["picks"].data_ptr())
        out = {"out": s["out"], "picks": s["picks"]}
    if rc != 0:
        raise RuntimeError("%s: refused" % op)
    return out


def run(s):
    if own:
        return _run_own(s)
    return {"attend": _attend, "evict": _evict, "summaries": _summaries, "blocks": _blocks}[s["case"]["op"]](s)


# ------------------------------------------------------------------------------------------- work and 64 bits

def work(case):
    H, nkv, hd = HEADS[case["heads"]]
    es = 4 if case["cache"] == "f32" else 2
    lens, B = _lens(case), case["B"]
    if case["op"] == "evict":
        n = 0
        for x in lens:
            kept = min(x, case["budget"])
            moved = (1 if x > kept else 0) if case["inplace"] else kept      # one token over budget: one slot changes hands
            n += nkv * (4 * x + moved * (2 * hd * es * 2 + 16))
        return {"bytes": n, "flops": 0}
    if case["op"] == "summaries":
        n = 0
        for x in lens:
            first = max(0, x - case["new"]) // case["block"] * case["block"]
            n += nkv * ((x - first) * hd * es + -(-(x - first) // case["block"]) * (hd + 4))
        return {"bytes": n, "flops": nkv * sum(lens) * hd}
    T, eq = case["T"], 4 if case["act"] == "f32" else 2
    by, fl = 2 * B * T * H * hd * eq, 0
    for x in lens:
        if case["op"] == "attend":
            by += nkv * (x + T) * 2 * hd * es + (8 * nkv * (x + T) if case["weights"] else 0)
            fl += 4 * hd * H * (T * x + T)
        else:
            nb = x // case["block"]
            keys = min(x + 1, case["n_sel"] * case["block"])
            by += nkv * (nb * (hd + 4) + min(x + T, T * keys) * 2 * hd * es) + 4 * T * nkv * case["n_sel"]
            fl += 4 * hd * H * T * keys + 2 * hd * H * T * nb
    return {"bytes": by, "flops": fl}


def _exact_row(q, k, v, ok):
    """[heads][tokens of a query] in float64: out and weights of one kv head's queries [n][hd] over keys [m][hd], `ok` [n][m]."""
    s = torch.einsum("nd,md->nm", q, k) / math.sqrt(q.shape[1])
    s = torch.where(ok, s, torch.full_like(s, -1e300))
    p = torch.softmax(s, 1) * ok
    return p @ v, p


def exact(case, seed):
    """The same outputs from the definitions, row by row, in 64 bits."""
    op = case["op"]
    if op == "evict":                               # nothing in it is computed: tokens are picked and moved
        return None
    H, nkv, hd = HEADS[case["heads"]]
    s = prepare(case, seed)
    B, G = case["B"], H // nkv
    lens = s["lens"].tolist()
    if op == "summaries":
        nb, block = s["codes"].shape[2], case["block"]
        out = torch.zeros(B, nkv, nb, hd, dtype=torch.float64, device="cuda")
        for b, n in enumerate(lens):
            lo = max(0, n - case["new"]) // block
            for i in range(lo, -(-n // block)):
                m = s["k"][b, :, i * block:min(n, (i + 1) * block)].double().mean(1)
                # a code is what the mean in 32 bits rounds to; the value it stands for is exact
                m32 = m.float()
                sc = (m32.abs().amax(1, keepdim=True) / 127.0)
                out[b, :, i] = torch.where(sc > 0, torch.round(m32 / sc), torch.zeros_like(m32)).double() * sc.double()
        return out
    T = case["T"]
    if B * T * nkv > 4096 and op == "blocks":
        return None
    out = torch.zeros(B, T, H, hd, dtype=torch.float64, device="cuda")
    if op == "attend":
        weights = s["weights"].double() if s["weights"] is not None else None
        parents = s["parents"].tolist() if s["parents"] is not None else None
        for b, n in enumerate(lens):
            ok = torch.zeros(T, n + T, dtype=torch.bool)
            for t in range(T):
                if parents is None:
                    ok[t, :n + t + 1] = True
                    continue
                if not -1 <= parents[b][t] < t:
                    continue
                ok[t, :n] = True
                at = t
                while at >= 0:
                    ok[t, n + at] = True
                    at = parents[b][at]
            ok = ok.cuda().repeat_interleave(G, 0)
            for h in range(nkv):
                o, p = _exact_row(s["q"][b, :, h * G:(h + 1) * G].reshape(T * G, hd).double(), s["k"][b, h, :n + T].double(), s["v"][b, h, :n + T].double(), ok)
                out[b, :, h * G:(h + 1) * G] = o.view(T, G, hd)
                if weights is not None:
                    weights[b, h, :n] += p[:, :n].sum(0)
                    weights[b, h, n:n + T] = p[:, n:].sum(0)
        return {"out": out} if weights is None else {"out": out, "weights": weights}
    picks = _pick(s)                                # whole numbers by definition: sums of products of 8-bit codes
    for b, n in enumerate(lens):
        for t in range(T):
            for h in range(nkv):
                p = picks[b, t, h].long()
                tok = (p[p >= 0][:, None] * case["block"] + torch.arange(case["block"], device="cuda")).view(-1)
                tok = tok[tok <= n + t]
                o, _ = _exact_row(s["q"][b, t, h * G:(h + 1) * G].double(), s["k"][b, h, tok].double(), s["v"][b, h, tok].double(),
                                  torch.ones(G, tok.numel(), dtype=torch.bool, device="cuda"))
                out[b, t, h * G:(h + 1) * G] = o
    return {"out": out, "picks": None}
