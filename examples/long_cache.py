"""Long-context decoding with the library's cache operators (include/ncm_b200.h, "operators on long key/value caches").

A small decoder of random weights -- two layers, 8 query heads over 2 kv heads of 64, a bf16 cache -- generates greedily from
one prompt in four ways:

* ``one by one``: every step attends to the whole cache with its one new token (ncmb_cache_attention);
* ``trees``: tokens are drafted from what followed the same token before, a tree of them is verified in one step, and the
  longest branch that the model agrees with is kept. The same text in fewer steps;
* ``budget``: the last tokens of the prompt add up attention weights, the cache is cut to a budget (ncmb_cache_evict) and held
  there, one token in, one token out;
* ``blocks``: mean keys of the prompt's blocks (ncmb_block_summaries), then every step reads the blocks its query picks
  (ncmb_block_attention).

    python examples/long_cache.py [--prompt 3000] [--new 48]

Products, norms and activations are the library's layer kernels; torch holds the memory and does what is left.
"""
import argparse
import importlib.util
import math
import os

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LAYERS, C, H, NKV, HD, HID, VOCAB = 2, 256, 8, 2, 64, 512, 512
BLOCK, N_SEL, BUDGET, RECENT = 32, 24, 512, 64


def load_library():
    spec = importlib.util.spec_from_file_location("graft_entry", os.path.join(ROOT, "__graft_entry__.py"))
    entry = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(entry)
    pkg = entry.load_package()
    return pkg.load_library(), pkg.capi


lib, capi = load_library()


class Cache:
    """One layer's keys and values of one row, token by token, and what the operators keep beside them."""

    def __init__(self, capacity):
        buf = torch.zeros(1, capacity, 2, NKV, HD, dtype=torch.bfloat16, device="cuda")
        self.k, self.v = (buf[:, :, i].permute(0, 2, 1, 3) for i in (0, 1))
        self.len = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.handle = capi.KVCache.of(self.k, self.v, self.len)
        self.weights = torch.zeros(1, NKV, capacity, device="cuda")
        self.pos = torch.zeros(1, NKV, capacity, dtype=torch.int32, device="cuda")
        nb = -(-capacity // BLOCK)
        self.codes, self.scales = torch.zeros(1, NKV, nb, HD, dtype=torch.int8, device="cuda"), torch.zeros(1, NKV, nb, device="cuda")


class Model:
    def __init__(self, seed, capacity):
        g = torch.Generator(device="cuda").manual_seed(seed)
        r = lambda *s, std: torch.randn(*s, device="cuda", generator=g) * std
        self.emb, self.head = r(VOCAB, C, std=0.3), r(VOCAB, C, std=1.0)
        self.w = [dict(n1=torch.ones(C, device="cuda"), qkv=r((H + 2 * NKV) * HD, C, std=1.6 / math.sqrt(C)), o=r(C, H * HD, std=1.0 / math.sqrt(H * HD)),
                       n2=torch.ones(C, device="cuda"), up=r(HID, C, std=1.0 / math.sqrt(C)), down=r(C, HID, std=1.0 / math.sqrt(HID))) for _ in range(LAYERS)]
        self.norm = torch.ones(C, device="cuda")
        a = torch.arange(capacity + 4096, device="cuda")[:, None] * 10000.0 ** (-torch.arange(HD // 2, device="cuda") / (HD // 2))
        self.cos, self.sin = a.cos(), a.sin()
        self.caches = [Cache(capacity) for _ in range(LAYERS)]
        self.held = 0                   # tokens in the caches
        self.seen = 0                   # tokens of the text so far

    def linear(self, x, w):
        y = torch.empty(x.shape[0], w.shape[0], device="cuda")
        lib.linear_fwd(x.data_ptr(), w.data_ptr(), None, y.data_ptr(), x.shape[0], w.shape[0], w.shape[1])
        return y

    def rms(self, x, w):
        y = torch.empty_like(x)
        lib.rmsnorm_fwd(x.data_ptr(), w.data_ptr(), y.data_ptr(), x.shape[0], C)
        return y

    def rotate(self, x, at):            # [T][heads][HD]
        c, s = self.cos[at][:, None], self.sin[at][:, None]
        a, b = x[..., :HD // 2], x[..., HD // 2:]
        return torch.cat([a * c - b * s, b * c + a * s], -1)

    def step(self, ids, parents=None, weights=False, blocks=False):
        """Logits of T new tokens, whose keys and values go to the slots behind the cached ones."""
        T = len(ids)
        depth = list(range(T))
        if parents is not None:
            for t in range(T):
                depth[t] = depth[parents[t]] + 1 if parents[t] >= 0 else 0
        at = torch.tensor(depth, device="cuda") + self.seen
        dpar = torch.tensor(parents, dtype=torch.int32, device="cuda") if parents is not None else None
        x = self.emb[torch.tensor(ids, device="cuda")].contiguous()
        for w, c in zip(self.w, self.caches):
            qkv = self.linear(self.rms(x, w["n1"]), w["qkv"]).view(T, H + 2 * NKV, HD)
            q = self.rotate(qkv[:, :H], at).contiguous()
            c.k[0, :, self.held:self.held + T] = self.rotate(qkv[:, H:H + NKV], at).transpose(0, 1)
            c.v[0, :, self.held:self.held + T] = qkv[:, H + NKV:].transpose(0, 1)
            out = torch.empty(T, H * HD, device="cuda")
            c.len.fill_(self.held)
            if blocks:
                rc = lib.ncmb_block_summaries(c.handle, T, c.len.data_ptr(), BLOCK, self.held, c.codes.data_ptr(), c.scales.data_ptr())
                rc |= lib.ncmb_block_attention(c.handle, q.data_ptr(), H * HD, out.data_ptr(), H * HD, capi.F32, H, T, BLOCK, c.codes.data_ptr(),
                                               c.scales.data_ptr(), N_SEL, 1, 2, 0.0, self.held, None)
            else:
                rc = lib.ncmb_cache_attention(c.handle, q.data_ptr(), H * HD, out.data_ptr(), H * HD, capi.F32, H, T, dpar.data_ptr() if parents is not None else None,
                                              0.0, self.held, c.weights.data_ptr() if weights else None)
            assert rc == 0
            x = x + self.linear(out, w["o"])
            h = self.linear(self.rms(x, w["n2"]), w["up"])
            lib.silu_fwd(h.data_ptr(), h.data_ptr(), h.numel())
            x = x + self.linear(h, w["down"])
        return self.linear(self.rms(x, self.norm), self.head)

    def take(self, n):
        self.held += n
        self.seen += n

    def prompt(self, ids, **kw):
        """In pieces of at most 256 tokens; the next token."""
        for i in range(0, len(ids), 256):
            piece = ids[i:i + 256]
            logits = self.step(piece, **kw)
            self.take(len(piece))
        return int(logits[-1].argmax())

    def evict(self, known):
        """Every layer's cache back to the budget; `known`: tokens of the last eviction."""
        n = min(self.held, BUDGET)
        dk, ds = (torch.tensor([v], dtype=torch.int32, device="cuda") for v in (known, self.seen))
        for c in self.caches:
            c.len.fill_(self.held)
            left = torch.empty(1, dtype=torch.int32, device="cuda")
            assert lib.ncmb_cache_evict(c.handle, c.handle, c.weights.data_ptr(), c.weights.data_ptr(), c.pos.data_ptr(), c.pos.data_ptr(), dk.data_ptr(),
                                        ds.data_ptr(), BUDGET, RECENT, self.held, left.data_ptr()) == 0
        self.held = n
        return n


def one_by_one(m, ids, new):
    tok, out = m.prompt(ids), []
    while len(out) < new:
        out.append(tok)
        tok = int(m.step([tok])[-1].argmax())
        m.take(1)
    return out, new


def draft(text, size, branches=3):
    """A tree over what followed the last token before: node 0 is that token; parents and tokens."""
    ids, parents, ends = [text[-1]], [-1], [(0, len(text) - 1)]
    follow = [i for i in range(len(text) - 2, -1, -1) if text[i] == text[-1]][:branches]
    for f in follow:
        at = 0
        for d in range(1, 1 + (size - 1) // branches):
            if f + d >= len(text) or len(ids) >= size:
                break
            same = [i for i in range(len(ids)) if parents[i] == at and ids[i] == text[f + d]]
            if same:
                at = same[0]
                continue
            ids.append(text[f + d])
            parents.append(at)
            at = len(ids) - 1
    return ids, parents


def trees(m, ids, new, size=16):
    tok, text, steps = m.prompt(ids), list(ids), 0
    text.append(tok)
    while len(text) - len(ids) < new + 1:
        nodes, parents = draft(text, size)
        pad = size - len(nodes)
        best = m.step(nodes + [0] * pad, parents + [-2] * pad).argmax(-1).tolist()
        path = [0]                      # the branch that the model agrees with
        while True:
            nxt = [i for i in range(len(nodes)) if parents[i] == path[-1] and nodes[i] == best[path[-1]]]
            if not nxt:
                break
            path.append(nxt[0])
        text += [nodes[i] for i in path[1:]] + [best[path[-1]]]
        for c in m.caches:              # its keys and values, one behind the other
            for x in (c.k, c.v):
                x[0, :, m.held:m.held + len(path)] = x[0, :, [m.held + i for i in path]]
        m.take(len(path))
        steps += 1
    return text[len(ids):len(ids) + new], steps


def budget(m, ids, new):
    m.prompt(ids[:-RECENT])
    tok, out = m.prompt(ids[-RECENT:], weights=True), []         # the last tokens look back: what is worth keeping
    known = m.evict(0)
    while len(out) < new:
        out.append(tok)
        tok = int(m.step([tok], weights=True)[-1].argmax())
        m.take(1)
        known = m.evict(known)
    return out, new


def blocks(m, ids, new):
    tok, out = m.prompt(ids), []
    for c in m.caches:
        c.len.fill_(m.held)
        assert lib.ncmb_block_summaries(c.handle, 0, None, BLOCK, m.held, c.codes.data_ptr(), c.scales.data_ptr()) == 0
    while len(out) < new:
        out.append(tok)
        tok = int(m.step([tok], blocks=True)[-1].argmax())
        m.take(1)
    return out, new


def run(prompt=3000, new=48, seed=0):
    """{way: (tokens, steps, tokens held at the end)}"""
    g = torch.Generator().manual_seed(seed)
    phrase = torch.randint(0, VOCAB, (97,), generator=g).tolist()          # a text that repeats itself, with slips
    ids = [phrase[i % 97] if torch.rand(1, generator=g) < 0.9 else int(torch.randint(0, VOCAB, (1,), generator=g)) for i in range(prompt)]
    got = {}
    for way in (one_by_one, trees, budget, blocks):
        m = Model(seed + 1, prompt + new + 64)
        out, steps = way(m, ids, new)
        got[way.__name__] = (out, steps, m.held)
    torch.cuda.synchronize()
    return got


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--prompt", type=int, default=3000)
    ap.add_argument("--new", type=int, default=48)
    a = ap.parse_args()
    got = run(a.prompt, a.new)
    ref = got["one_by_one"][0]
    for way, (out, steps, held) in got.items():
        same = sum(x == y for x, y in zip(out, ref))
        print("%-11s %3d tokens in %3d steps, %5d tokens held, %3d of %d the same as one by one; first: %s" % (way, len(out), steps, held, same, len(ref), out[:8]))
