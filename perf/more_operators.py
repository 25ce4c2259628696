"""Operators of beam search over a paged key/value cache, as cases that can be timed and compared.

* ``rope``    -- ``ncmb_rope``: rotary positions, halves or neighbouring pairs of dims, all or the first dims of a head, with the
  scalings for long contexts, forward and back (which is also the gradient);
* ``append``  -- ``ncmb_paged_append``: new tokens' keys, rotated on the way, and values into the pages of their rows, queries rotated too;
* ``attend``  -- ``ncmb_paged_attention``: one new token a row, or a short run, attends to the row's pages;
* ``select``  -- ``ncmb_beam_select``: the best continuations of every group of beams over beams and vocabulary;
* ``reorder`` -- ``ncmb_paged_reorder``: rows continue from the beams that were selected: full pages are shared, begun ones copied.

Shapes of heads, layers and vocabularies are this repository's decoder and generator configurations (12 x 64 with 12 layers and 50257
words, 14 over 2 x 64 with 24 layers and 151936 words, 16 over 4 x 64 with 24 layers and 16384 codes) and the generic 32 over 8 x 128.
"""
import functools
import math

import torch

own = False

# query heads, kv heads, head dim, layers, words
HEADS = {"gpt2": (12, 12, 64, 12, 50257), "qwen": (14, 2, 64, 24, 151936), "box": (16, 4, 64, 24, 16384), "wide": (32, 8, 128, 32, 128000)}
FMAX = torch.finfo(torch.float32).max


# ------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # queries and keys of a decode step of five users, the smallest call: all latency
        {"name": "rope_step_qwen_5x1", "op": "rope", "heads": "qwen", "act": "f32", "B": 5, "T": 1, "layout": "halves", "dims": 64, "scaling": "plain",
         "theta": 1000000.0, "far": 30000, "inverse": False},
        # prompts in bf16, neighbouring pairs in the first half of each head, base stretched for four times the length
        {"name": "rope_prompt_wide_8x4000", "op": "rope", "heads": "wide", "act": "bf16", "B": 8, "T": 4000, "layout": "pairs", "dims": 64, "scaling": "base",
         "theta": 10000.0, "far": 9000, "inverse": False},
        # gradients of a training batch rotated back, far positions, frequencies stretched by parts
        {"name": "rope_back_box_3x4097", "op": "rope", "heads": "box", "act": "f32", "B": 3, "T": 4097, "layout": "halves", "dims": 64, "scaling": "parts",
         "theta": 500000.0, "far": 900000, "inverse": True},
        # a decode step of a batch: one token a row into pages of 16
        {"name": "append_step_qwen_48", "op": "append", "heads": "qwen", "cache": "bf16", "act": "f32", "layout": "token", "rope": "halves", "dims": 64, "B": 48, "len": 5000,
         "new": 1, "ragged": True, "page": 16},
        # pieces of prompts of all lengths, one behind the other, into pages of 64
        {"name": "append_prompt_wide_16x2001", "op": "append", "heads": "wide", "cache": "bf16", "act": "bf16", "layout": "head", "rope": "pairs", "dims": 128, "B": 16,
         "len": 900, "new": 2001, "ragged": True, "page": 64},
        # one interactive completion of the GPT-2 shape, fp32 cache
        {"name": "attend_gpt2_1x701", "op": "attend", "heads": "gpt2", "cache": "f32", "act": "f32", "layout": "token", "B": 1, "T": 1, "len": 701, "ragged": False, "page": 16},
        # a decode step of a batch of the Qwen2 shape, rows of all lengths, one of them new
        {"name": "attend_qwen_48x6000", "op": "attend", "heads": "qwen", "cache": "bf16", "act": "f32", "layout": "token", "B": 48, "T": 1, "len": 6000, "ragged": True, "page": 16},
        # a server's step over long rows
        {"name": "attend_wide_64x16000", "op": "attend", "heads": "wide", "cache": "bf16", "act": "bf16", "layout": "head", "B": 64, "T": 1, "len": 16000, "ragged": True,
         "page": 64},
        # four beams of one user, two candidates a beam
        {"name": "select_gpt2_1x4", "op": "select", "heads": "gpt2", "act": "f32", "B": 1, "beams": 4, "n_out": 8, "first": False, "done": False},
        # eight beams of a batch of the largest vocabulary, some of them at their end
        {"name": "select_qwen_32x8", "op": "select", "heads": "qwen", "act": "f32", "B": 32, "beams": 8, "n_out": 8, "first": False, "done": True},
        # four users with four beams, 24 layers
        {"name": "reorder_qwen_4x4", "op": "reorder", "heads": "qwen", "cache": "bf16", "layout": "token", "B": 4, "beams": 4, "len": 5000, "page": 16},
        # a batch of eight beams each, 32 layers, pages of 64
        {"name": "reorder_wide_16x8", "op": "reorder", "heads": "wide", "cache": "bf16", "layout": "head", "B": 16, "beams": 8, "len": 4000, "page": 64},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        c = {"op": rng.choice(["rope", "append", "attend", "attend", "select", "select", "reorder"]), "heads": rng.choice(list(HEADS))}
        H, nkv, hd, layers, V = HEADS[c["heads"]]
        if c["op"] == "rope":
            c.update(act=rng.choice(["f32", "bf16"]), B=_log(rng, 1, 64), T=_log(rng, 1, 5000), layout=rng.choice(["halves", "pairs"]), dims=2 * rng.randint(2, hd // 2),
                     scaling=rng.choice(["plain", "linear", "base", "parts"]), theta=rng.choice([10000.0, 500000.0, 1000000.0]), far=_log(rng, 1, 1000000),
                     inverse=rng.random() < 0.4)
            if rng.random() < 0.5:
                c["dims"] = rng.choice([hd, hd // 2])
            if c["B"] * c["T"] * (H + nkv) * hd <= 1.6e8:
                return c
            continue
        if c["op"] == "select":
            c.update(act=rng.choice(["f32", "f32", "bf16"]), B=_log(rng, 1, 64), beams=_log(rng, 1, 32), first=rng.random() < 0.2, done=rng.random() < 0.4)
            c["n_out"] = rng.choice([c["beams"], 2 * c["beams"], _log(rng, 1, 64)])
            if c["B"] * c["beams"] * V <= 3.9e7:
                return c
            continue
        c.update(cache=rng.choice(["f32", "bf16", "bf16"]), layout=rng.choice(["token", "head"]), page=rng.choice([8, 16, 32, 64, 128, 256]))
        es = 4 if c["cache"] == "f32" else 2
        if c["op"] == "reorder":
            c.update(B=_log(rng, 1, 32), beams=rng.randint(1, 16), len=_log(rng, 1, 8000))
            if 2 * layers * nkv * hd * es * c["page"] * (c["B"] * c["beams"] + 8) <= 1.5e9:
                return c
            continue
        c.update(act="f32" if c["cache"] == "f32" else rng.choice(["f32", "bf16"]), B=_log(rng, 1, 64), len=_log(rng, 1, 16000), ragged=rng.random() < 0.6)
        if c["op"] == "append":
            c.update(rope=rng.choice(["halves", "pairs", "none"]), dims=rng.choice([hd, hd // 2, 2 * rng.randint(2, hd // 2)]), new=rng.choice([1, _log(rng, 2, 3000)]))
            if c["B"] * c["new"] * (H + 2 * nkv) * hd <= 1.6e8 and 2 * c["B"] * nkv * (c["len"] + c["new"]) * hd * es <= 1.5e9:
                return c
        else:
            c["T"] = rng.choice([1, 1, 1, rng.randint(2, 8)])
            if 2 * c["B"] * nkv * c["len"] * hd * es <= 1.7e9:
                return c


# ------------------------------------------------------------------------------------------- inputs

def _lens(case):
    """Cached tokens of each row: the stated length, or lengths from nothing up to it."""
    B, n = case["B"] * case.get("beams", 1), case["len"]
    if case["op"] == "reorder":                       # beams of a group have taken as many steps
        return [max(0, n - 97 * (b // case["beams"])) for b in range(B)]
    if not case["ragged"] or B == 1:
        return [n] * B
    out = [min(n, max(1, n * (16 + (b * 37 + 11) % 48) // 63)) for b in range(B)]
    out[0], out[1] = n, 0                             # the longest, and a row that has just been opened
    return out


def _news(case):
    """New tokens of each row of an append."""
    if not case["ragged"] or case["new"] == 1:
        return [case["new"]] * case["B"]
    return [max(1, case["new"] * (7 + (b * 29 + 5) % 57) // 63) for b in range(case["B"])]


def _type(name):
    return torch.float32 if name == "f32" else torch.bfloat16


def _pool(case, n_pages, layers, g):
    """Keys and values [layer][page][kv head][slot][hd], whatever their order in memory; slots hold what earlier texts left."""
    H, nkv, hd = HEADS[case["heads"]][:3]
    dt, page = _type(case["cache"]), case["page"]
    if case["layout"] == "token":                     # a page: [slot][keys | values of all heads]
        buf = torch.randn(layers, n_pages, page, 2, nkv, hd, device="cuda", dtype=dt, generator=g)
        return buf[:, :, :, 0].transpose(2, 3), buf[:, :, :, 1].transpose(2, 3)
    buf = torch.randn(2, layers, n_pages, nkv, page, hd, device="cuda", dtype=dt, generator=g)
    return buf[0], buf[1]


def _turns(case):
    """Positions' frequencies, radians a position in 64 bits, for a plan."""
    n, theta = case["dims"], case.get("theta", 10000.0)
    scaling, factor, trained, low, high = case.get("scaling", "plain"), 4.0, 8192.0, 1.0, 4.0
    if scaling == "base" and n > 2:
        theta *= factor ** (n / (n - 2.0))
    f = [theta ** (-2.0 * i / n) for i in range(n // 2)]
    if scaling == "linear":
        f = [x / factor for x in f]
    if scaling == "parts":
        r = [min(1.0, max(0.0, (trained * x / (2 * math.pi) - low) / (high - low))) for x in f]
        f = [x * (y + (1 - y) / factor) for x, y in zip(f, r)]
    return f


def _magnitude(case):
    return 0.1 * math.log(4.0) + 1.0 if case.get("scaling") == "parts" else 1.0


def prepare(case, seed):
    H, nkv, hd, layers, V = HEADS[case["heads"]]
    g = torch.Generator(device="cuda").manual_seed(int(seed) & 0x7fffffff)
    op, B = case["op"], case["B"]
    s = {"case": case}
    r = lambda *shape: torch.randn(*shape, device="cuda", generator=g)
    if op in ("rope", "append"):
        s["freq"] = torch.tensor(_turns(case), dtype=torch.float64, device="cuda")
        s["magnitude"] = _magnitude(case)
    if op == "rope":
        # queries and keys of a projection, the values' columns beside them
        s["x"] = r(B, case["T"], H + 2 * nkv, hd).to(_type(case["act"]))[:, :, :H + nkv]
        s["y"] = torch.empty(B, case["T"], H + nkv, hd, device="cuda", dtype=s["x"].dtype)
        first = torch.randint(0, case["far"] + 1, (B, 1), device="cuda", generator=g)
        s["pos"] = (first + torch.arange(case["T"], device="cuda")).int()
        return s
    if op == "select":
        K = case["beams"]
        # a few words stand out from the others
        x = r(B * K, V).mul_(2)
        x += 6 * r(B * K, V).clamp_(min=2.5).sub_(2.5)
        s["logits"] = x.to(_type(case["act"]))
        s["scores"] = -20.0 - 6 * torch.rand(B, K, device="cuda", generator=g)
        if case["first"]:                             # a group's beams are still the same: one of them counts
            s["scores"][:, 1:] = float("-inf")
        s["done"] = (torch.rand(B, K, device="cuda", generator=g) < 0.2).int() if case["done"] else None
        s["eos"] = 2
        n = case["n_out"]
        s["scores_out"], s["parents"], s["tokens"] = torch.empty(B, n, device="cuda"), torch.empty(B, n, dtype=torch.int32, device="cuda"), torch.empty(B, n, dtype=torch.int32, device="cuda")
        s["done_out"] = torch.empty(B, n, dtype=torch.int32, device="cuda")
        return s
    lens, page = _lens(case), case["page"]
    rows = len(lens)
    news = _news(case) if op == "append" else [case.get("T", 1)] * rows
    need = [(n + t - 1) // page + 1 for n, t in zip(lens, news)]       # pages up to the one of the last new token
    width = max(need) + 2
    if op == "reorder":
        # the beams of a group share their full pages, each has a begun page and one in reserve
        K = case["beams"]
        full = [lens[b * K] // page for b in range(B)]
        # of the shared pages, which are not touched, a few stand for all
        shared = 8
        n_pages = shared + 2 * rows
        perm = (torch.randperm(n_pages - shared, device="cuda", generator=g) + shared).int()
        table = torch.randint(0, shared, (B, 1, width), device="cuda", generator=g).int().expand(B, K, width).reshape(rows, width).clone()
        col, at = torch.arange(width, device="cuda"), torch.tensor(full, device="cuda").repeat_interleave(K)[:, None]
        table = torch.where(col == at, perm[:rows, None], torch.where(col == at + 1, perm[rows:, None], torch.where(col > at, -1, table))).int()
        s["k"], s["v"] = _pool(case, n_pages, layers, g)
        s["parents"] = torch.randint(0, K, (B, K), device="cuda", generator=g).int()
        s["table2"], s["lens2"] = torch.empty_like(table), torch.empty(rows, dtype=torch.int32, device="cuda")
    else:
        n_pages = sum(need) + 3
        perm = torch.randperm(n_pages, device="cuda", generator=g)
        col, count = torch.arange(width, device="cuda"), torch.tensor(need, device="cuda")
        first = count.cumsum(0) - count
        table = torch.where(col < count[:, None], perm[(first[:, None] + col).clamp(max=n_pages - 1)], -1).int()
        k, v = _pool(case, n_pages, 1, g)
        s["k"], s["v"] = k[0], v[0]
    s["table"], s["lens"] = table, torch.tensor(lens, dtype=torch.int32, device="cuda")
    s["max_len"] = max(lens)
    if op == "append":
        total = sum(news)
        dt = _type(case["act"])
        s["qkv"] = r(total, H + 2 * nkv, hd).to(dt)
        s["q_out"] = torch.empty(total, H, hd, device="cuda", dtype=dt)
        s["start"] = torch.tensor([0] + news, device="cuda").cumsum(0).int()
    if op == "attend":
        dt = _type(case["act"])
        s["q"] = r(rows, case["T"], H, hd).mul_(1.5).to(dt)
        s["out"] = torch.empty(rows, case["T"], H, hd, device="cuda", dtype=dt)
    return s


# ------------------------------------------------------------------------------------------- plain forms

def _rotate(x, pos, freq, magnitude, pairs, inverse=False):
    """x [...][heads][hd], pos [...]: the first 2 len(freq) dims rotated, in fp32; angles in 64 bits."""
    n = 2 * freq.numel()
    a = pos.double()[..., None] * freq
    c, sn = (a.cos() * magnitude).float()[..., None, :], (a.sin() * (-magnitude if inverse else magnitude)).float()[..., None, :]
    x = x.float()
    if pairs:
        p, q = x[..., 0:n:2], x[..., 1:n:2]
        y = torch.stack([p * c - q * sn, q * c + p * sn], -1).flatten(-2)
    else:
        p, q = x[..., :n // 2], x[..., n // 2:n]
        y = torch.cat([p * c - q * sn, q * c + p * sn], -1)
    return torch.cat([y, x[..., n:]], -1)


def _rope(s):
    case = s["case"]
    return _rotate(s["x"], s["pos"], s["freq"], s["magnitude"], case["layout"] == "pairs", case["inverse"]).to(s["x"].dtype)


def _append(s):
    case = s["case"]
    H, nkv, hd = HEADS[case["heads"]][:3]
    page, x = case["page"], s["qkv"]
    i = torch.arange(x.shape[0], device="cuda")
    row = torch.searchsorted(s["start"].long(), i, right=True) - 1
    at = s["lens"].long()[row] + i - s["start"].long()[row]
    q, k, v = x[:, :H].float(), x[:, H:H + nkv].float(), x[:, H + nkv:]
    if case["rope"] != "none":
        q, k = (_rotate(y, at, s["freq"], s["magnitude"], case["rope"] == "pairs") for y in (q, k))
    to = s["table"].long()[row, at // page]
    s["k"][to, :, at % page] = k.to(s["k"].dtype)
    s["v"][to, :, at % page] = v.to(s["v"].dtype)
    return {"q": q.to(x.dtype), "k": s["k"], "v": s["v"]}


def _attend(s):
    case = s["case"]
    H, nkv, hd = HEADS[case["heads"]][:3]
    B, T, G = case["B"], case["T"], H // nkv
    table = s["table"].long().clamp(min=0)
    cap = table.shape[1] * case["page"]
    k, v = (s[x][table].transpose(1, 2).reshape(B, nkv, cap, hd).float() for x in "kv")
    q = s["q"].float().view(B, T, nkv, G, hd).permute(0, 2, 1, 3, 4).reshape(B, nkv, T * G, hd)
    here = s["lens"].long()[:, None] + torch.arange(T, device="cuda")                           # [B][T]
    seen = torch.arange(cap, device="cuda") <= here[:, :, None]                                 # [B][T][cap]
    sc = (q @ k.transpose(2, 3)).view(B, nkv, T, G, cap) * (1.0 / math.sqrt(hd))
    sc = sc.masked_fill(~seen[:, None, :, None], float("-inf"))
    e = torch.exp(sc - sc.amax(-1, keepdim=True))
    p = (e / e.sum(-1, keepdim=True)).view(B, nkv, T * G, cap)
    v = v.masked_fill((torch.arange(cap, device="cuda") > here[:, -1:])[:, None, :, None], 0.0)
    return (p @ v).view(B, nkv, T, G, hd).permute(0, 2, 1, 3, 4).reshape(B, T, H, hd).to(s["q"].dtype)


def _select(s):
    """Scores in 64 bits: where two continuations are near one another, the order must not hang on how a sum was rounded. A beam's own
    continuations are in the order of their logits."""
    case = s["case"]
    B, K, n = case["B"], case["beams"], case["n_out"]
    x = s["logits"].float().nan_to_num(nan=float("-inf"), posinf=FMAX, neginf=float("-inf")).view(B, K, -1)
    V = x.shape[2]
    if s["done"] is not None:                                                                   # goes on with its end, at no cost
        end = torch.where(torch.arange(V, device="cuda") == s["eos"], 0.0, float("-inf"))
        x = torch.where((s["done"] != 0)[:, :, None], end, x)
    words = x.sort(dim=2, descending=True, stable=True).indices[:, :, :n]
    x = x.double()
    top = x.amax(2, keepdim=True)
    top = top.masked_fill(top == float("-inf"), 0.0)
    total = top + torch.exp(x - top).sum(2, keepdim=True).clamp_(min=5e-324).log()              # of a row of nothing: all stays -infinity
    score = (s["scores"].double()[:, :, None] + (x.gather(2, words) - total)).flatten(1)
    best, at = (y[:, :n] for y in score.sort(dim=1, descending=True, stable=True))
    parents, tokens = at // words.shape[2], words.flatten(1).gather(1, at)
    done = tokens == s["eos"]
    if s["done"] is not None:
        done |= s["done"].gather(1, parents) != 0
    return {"scores": best.float(), "parents": parents.int(), "tokens": tokens.int(), "done": done.int()}


def _reorder(s):
    case = s["case"]
    B, K, page = case["B"], case["beams"], case["page"]
    par, lens, table = s["parents"].long(), s["lens"].long().view(B, K), s["table"].long().view(B, K, -1)
    width = table.shape[2]
    beam = torch.arange(K, device="cuda")
    again = ((par[:, :, None] == par[:, None, :]) & (beam[None, :] < beam[:, None])).any(2)     # an earlier beam has this parent
    alive = (par[:, :, None] == beam).any(1)
    free = alive.long().sort(dim=1, stable=True).indices                                        # beams without children first, ascending
    owner = torch.where(again, free.gather(1, (again.long().cumsum(1) - 1).clamp(min=0)), par)  # whose own pages a beam goes on with
    n = lens.gather(1, par)
    tp, to = (n // page)[:, :, None], (lens.gather(1, owner) // page)[:, :, None]
    of = lambda rows: table.gather(1, rows[:, :, None].expand(B, K, width))
    col = torch.arange(width, device="cuda")
    src = col + to - tp
    mine = torch.where(src < width, of(owner).gather(2, src.clamp(0, width - 1)), -1)
    s["table2"].copy_(torch.where(col < tp, of(par), mine).view(B * K, width))
    s["lens2"].copy_(n.view(-1))
    a, b = of(par).gather(2, tp).view(-1), of(owner).gather(2, to).view(-1)
    begun = (torch.arange(page, device="cuda") < (n % page).view(-1, 1))[None, :, None, :, None]
    s["k"].index_copy_(1, b, torch.where(begun, s["k"][:, a], s["k"][:, b]))
    s["v"].index_copy_(1, b, torch.where(begun, s["v"][:, a], s["v"][:, b]))
    return {"table": s["table2"], "len": s["lens2"], "k": s["k"], "v": s["v"]}


# ------------------------------------------------------------------------------------------- the framework's

@functools.lru_cache(maxsize=1)
def _library():
    import __graft_entry__
    pkg = __graft_entry__.load_package()
    return pkg.load_library(), pkg.capi


def _plan(s):
    """The rotation's plan, which a program makes once."""
    if "plan" not in s:
        lib, capi = _library()
        case = s["case"]
        kinds = {"plain": capi.ROPE_PLAIN, "linear": capi.ROPE_LINEAR, "base": capi.ROPE_BASE, "parts": capi.ROPE_PARTS}
        s["plan"] = capi.Rope()
        layout = capi.ROPE_PAIRS if "pairs" in (case.get("rope"), case["layout"]) else capi.ROPE_HALVES
        if lib.ncmb_rope_plan(s["plan"], case["dims"], layout, case.get("theta", 10000.0), kinds[case.get("scaling", "plain")], 4.0, 8192.0, 1.0, 4.0, s["magnitude"]) != 0:
            raise RuntimeError("no plan")
    return s["plan"]


def _handle(s):
    """The library's view of a paged cache, which a program makes when it allocates one."""
    if "handle" not in s:
        k, v = (s[x][0] if s[x].dim() == 5 else s[x] for x in "kv")
        s["handle"] = _library()[1].PagedCache.of(k, v, s["table"], s["lens"])
    return s["handle"]


def _run_own(s):
    lib, capi = _library()
    case, op = s["case"], s["case"]["op"]
    H, nkv, hd, layers, V = HEADS[case["heads"]]
    act = capi.BF16 if case.get("act") == "bf16" else capi.F32
    if op == "rope":
        x, y = s["x"], s["y"]
        rc = lib.ncmb_rope(_plan(s), x.data_ptr(), capi.strides(x, 3), y.data_ptr(), capi.strides(y, 3), act, case["B"], case["T"], H + nkv, hd, s["pos"].data_ptr(),
                           int(case["inverse"]))
        out = y
    elif op == "append":
        x, es = s["qkv"], s["qkv"].element_size()
        p, ld = x.data_ptr(), (H + 2 * nkv) * hd
        rc = lib.ncmb_paged_append(_handle(s), _plan(s) if case["rope"] != "none" else None, p, ld, s["q_out"].data_ptr(), H * hd, H, p + H * hd * es, ld,
                                   p + (H + nkv) * hd * es, ld, act, x.shape[0], s["start"].data_ptr(), None)
        out = {"q": s["q_out"], "k": s["k"], "v": s["v"]}
    elif op == "attend":
        rc = lib.ncmb_paged_attention(_handle(s), s["q"].data_ptr(), H * hd, s["out"].data_ptr(), H * hd, act, H, case["T"], None, 0.0, s["max_len"])
        out = s["out"]
    elif op == "select":
        done = s["done"].data_ptr() if s["done"] is not None else None
        rc = lib.ncmb_beam_select(s["logits"].data_ptr(), V, act, case["B"], case["beams"], V, s["scores"].data_ptr(), done, s["eos"], case["n_out"],
                                  s["scores_out"].data_ptr(), s["parents"].data_ptr(), s["tokens"].data_ptr(), s["done_out"].data_ptr())
        out = {"scores": s["scores_out"], "parents": s["parents"], "tokens": s["tokens"], "done": s["done_out"]}
    else:
        rc = lib.ncmb_paged_reorder(_handle(s), case["beams"], s["parents"].data_ptr(), layers, s["k"].stride(0), s["table2"].data_ptr(), s["lens2"].data_ptr(), None)
        out = {"table": s["table2"], "len": s["lens2"], "k": s["k"], "v": s["v"]}
    if rc != 0:
        raise RuntimeError("%s: refused" % op)
    return out


def run(s):
    if own:
        return _run_own(s)
    return {"rope": _rope, "append": _append, "attend": _attend, "select": _select, "reorder": _reorder}[s["case"]["op"]](s)


# ------------------------------------------------------------------------------------------- work and 64 bits

def work(case):
    H, nkv, hd, layers, V = HEADS[case["heads"]]
    ea, ec = 4 if case.get("act") == "f32" else 2, 4 if case.get("cache") == "f32" else 2
    op, B = case["op"], case["B"]
    if op == "rope":
        n = B * case["T"] * (H + nkv) * hd
        return {"bytes": 2 * n * ea, "flops": 3 * n}
    if op == "select":
        n = B * case["beams"] * V
        return {"bytes": n * ea, "flops": 4 * n}
    if op == "reorder":                               # of a group's beams, (1 - 1 / K)^K have no children on the average
        K = case["beams"]
        lens = _lens(case)
        share = (1 - 1 / K) ** K if K > 1 else 0.0
        begun = sum(n % case["page"] for n in lens) * share
        return {"bytes": int(4 * begun * layers * nkv * hd * ec) + 8 * sum(n // case["page"] + 1 for n in lens), "flops": 0}
    if op == "append":
        n = sum(_news(case))
        return {"bytes": n * hd * (2 * H * ea + 2 * nkv * (ea + ec)), "flops": 3 * n * (H + nkv) * hd}
    T = case["T"]
    lens = _lens(case)
    return {"bytes": 2 * B * T * H * hd * ea + sum((n + T) * 2 * nkv * hd * ec for n in lens), "flops": sum(4 * H * hd * T * (n + T) for n in lens)}


def _turned(x, at, freq, m, pairs, back):
    """float64, by complex numbers: a pair of dims is one, a rotation a product."""
    n = 2 * freq.numel()
    x = x.double()
    z = torch.complex(x[..., 0:n:2].contiguous(), x[..., 1:n:2].contiguous()) if pairs else torch.complex(x[..., :n // 2].contiguous(), x[..., n // 2:n].contiguous())
    a = (at.double()[..., None] * freq)[..., None, :]
    z = z * torch.polar(torch.full_like(a, m), -a if back else a)
    y = x.clone()
    if pairs:
        y[..., 0:n:2], y[..., 1:n:2] = z.real, z.imag
    else:
        y[..., :n // 2], y[..., n // 2:n] = z.real, z.imag
    return y


def exact(case, seed):
    """The same outputs from the definitions, row by row, in 64 bits."""
    op = case["op"]
    if op == "reorder":                               # nothing in it is computed: pages are passed on and copied
        return None
    s = prepare(case, seed)
    H, nkv, hd = HEADS[case["heads"]][:3]
    if op == "rope":
        return torch.stack([_turned(s["x"][b], s["pos"][b], s["freq"], s["magnitude"], case["layout"] == "pairs", case["inverse"]) for b in range(case["B"])])
    if op == "select":
        B, K, n = case["B"], case["beams"], case["n_out"]
        scores = torch.empty(B, n, dtype=torch.float64, device="cuda")
        for b in range(B):
            rows = torch.log_softmax(s["logits"][b * K:(b + 1) * K].double(), 1) + s["scores"][b].double()[:, None]
            for k in range(K):
                if s["done"] is not None and s["done"][b, k]:
                    rows[k] = float("-inf")
                    rows[k, s["eos"]] = s["scores"][b, k].double()
            scores[b] = torch.topk(rows.flatten(), n).values
        return {"scores": scores, "parents": None, "tokens": None, "done": None}
    page, lens, table = case["page"], s["lens"].tolist(), s["table"].long()
    if op == "append":
        news = _news(case)
        k, v, q, i = s["k"].double(), s["v"].double(), torch.empty(sum(news), H, hd, dtype=torch.float64, device="cuda"), 0
        for b, t in enumerate(news):
            x, at = s["qkv"][i:i + t], torch.arange(lens[b], lens[b] + t, device="cuda")
            turn = (lambda y: y.double()) if case["rope"] == "none" else (lambda y: _turned(y, at, s["freq"], s["magnitude"], case["rope"] == "pairs", False))
            q[i:i + t] = turn(x[:, :H])
            to = table[b, at // page]
            k[to, :, at % page], v[to, :, at % page] = turn(x[:, H:H + nkv]), x[:, H + nkv:].double()
            i += t
        return {"q": q, "k": k, "v": v}
    T, G = case["T"], H // nkv
    out = torch.empty(case["B"], T, H, hd, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        pages = table[b, :(n + T - 1) // page + 1]
        k, v = (s[x][pages].permute(1, 0, 2, 3).reshape(nkv, -1, hd)[:, :n + T].double() for x in "kv")
        for t in range(T):
            q = s["q"][b, t].double().view(nkv, G, hd)
            p = torch.softmax(torch.einsum("hgd,hmd->hgm", q, k[:, :n + t + 1]) / math.sqrt(hd), -1)
            out[b, t] = torch.einsum("hgm,hmd->hgd", p, v[:, :n + t + 1]).reshape(H, hd)
    return out
