"""Beam search with the library's operators on paged caches (include/ncm_b200.h, "paged caches and beams").

A small decoder of random weights -- two layers, 8 query heads over 2 kv heads of 64 -- continues a few prompts with several beams each. Keys and values
stand in pages of one pool; the beams of a prompt share its pages and what they have had in common since. A step is

    ncmb_paged_append      rotates queries and keys and stores keys and values,      } per
    ncmb_paged_attention   attends to the rows' pages,                               } layer
    ncmb_beam_select       picks the best continuations of every group of beams,
    ncmb_paged_reorder     lets every row go on as the beam that it continues,

and nothing of it is read back before the end. Every row has pages in reserve for the steps to come; which of them a row owns changes as beams are
dropped and continued. A beam that has ended stays with its score.

    python examples/beam_search.py [--prompts 3] [--beams 4] [--new 24] [--cache bf16]

Products, norms and activations are the library's layer kernels; torch holds the memory and does what is left.
"""
import argparse
import importlib.util
import math
import os

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LAYERS, C, H, NKV, HD, HID, VOCAB = 2, 256, 8, 2, 64, 512, 500
PAGE, EOS = 16, 7


def load_library():
    spec = importlib.util.spec_from_file_location("graft_entry", os.path.join(ROOT, "__graft_entry__.py"))
    entry = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(entry)
    pkg = entry.load_package()
    return pkg.load_library(), pkg.capi


lib, capi = load_library()


class Weights:
    def __init__(self, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        r = lambda *s, std: torch.randn(*s, device="cuda", generator=g) * std
        self.emb, self.head = r(VOCAB, C, std=0.3), r(VOCAB, C, std=0.2)
        self.layers = [dict(qkv=r((H + 2 * NKV) * HD, C, std=1.6 / math.sqrt(C)), o=r(C, H * HD, std=1.0 / math.sqrt(H * HD)), up=r(HID, C, std=1.0 / math.sqrt(C)),
                            down=r(C, HID, std=1.0 / math.sqrt(HID))) for _ in range(LAYERS)]
        self.one = torch.ones(C, device="cuda")


class Decoder:
    """`groups` prompts with `beams` rows each."""

    def __init__(self, weights, groups, beams, longest, new, cache):
        self.w, self.groups, self.beams, self.rows = weights, groups, beams, groups * beams
        own = -(-(new + PAGE) // PAGE) + 1                        # a row's begun page and its reserve
        shared = -(-longest // PAGE)
        self.max_pages = shared + own + 1
        n_pages = groups * shared + self.rows * own
        self.pool = torch.zeros(2, LAYERS, n_pages, NKV, PAGE, HD, dtype=cache, device="cuda")
        self.table, self.table2 = (torch.full((self.rows, self.max_pages), -1, dtype=torch.int32, device="cuda") for _ in range(2))
        self.len, self.len2 = (torch.zeros(self.rows, dtype=torch.int32, device="cuda") for _ in range(2))
        pages = torch.arange(n_pages, dtype=torch.int32, device="cuda")
        # row 0 of a group holds the prompt, then its own pages; the others have own pages alone until they go on as row 0
        mine = pages[groups * shared:].view(self.rows, own)
        self.table[:, :own] = mine
        self.table[::beams, :shared] = pages[:groups * shared].view(groups, shared)
        self.table[::beams, shared:shared + own] = mine[::beams]
        # views of layer l with either table: all rows, or the groups' first ones (for the prompts)
        self.caches = [[capi.PagedCache.of(self.pool[0, l], self.pool[1, l], t, n) for l in range(LAYERS)] for t, n in ((self.table, self.len), (self.table2, self.len2))]
        self.first_len = torch.zeros(groups, dtype=torch.int32, device="cuda")
        self.firsts = [capi.PagedCache.of(self.pool[0, l], self.pool[1, l], self.table[::beams], self.first_len) for l in range(LAYERS)]
        self.plan = capi.Rope()
        assert lib.ncmb_rope_plan(self.plan, HD, capi.ROPE_HALVES, 10000.0, capi.ROPE_PLAIN, 1.0, 0.0, 0.0, 0.0, 1.0) == 0
        self.at = 0                                               # which of the tables holds

    def linear(self, x, w):
        y = torch.empty(x.shape[0], w.shape[0], device="cuda")
        lib.linear_fwd(x.data_ptr(), w.data_ptr(), None, y.data_ptr(), x.shape[0], w.shape[0], w.shape[1])
        return y

    def rms(self, x):
        y = torch.empty_like(x)
        lib.rmsnorm_fwd(x.data_ptr(), self.w.one.data_ptr(), y.data_ptr(), x.shape[0], C)
        return y

    def forward(self, tokens, caches, rows):
        """Logits of int64 tokens [rows * T], T new ones of every row of the caches."""
        x = self.w.emb[tokens].contiguous()
        n, ld = x.shape[0], (H + 2 * NKV) * HD
        for w, c in zip(self.w.layers, caches):
            qkv = self.linear(self.rms(x), w["qkv"])
            p, out = qkv.data_ptr(), torch.empty(n, H * HD, device="cuda")
            rc = lib.ncmb_paged_append(c, self.plan, p, ld, p, ld, H, p + H * HD * 4, ld, p + (H + NKV) * HD * 4, ld, capi.F32, n, None, None)
            rc |= lib.ncmb_paged_attention(c, p, ld, out.data_ptr(), H * HD, capi.F32, H, n // rows, None, 0.0, 0)
            assert rc == 0
            x = x + self.linear(out, w["o"])
            h = self.linear(self.rms(x), w["up"])
            lib.silu_fwd(h.data_ptr(), h.data_ptr(), h.numel())
            x = x + self.linear(h, w["down"])
        return self.linear(self.rms(x), self.w.head)

    def select(self, logits, beams, scores, done):
        G, K = self.groups, self.beams
        out = torch.empty(G, K, device="cuda"), *(torch.empty(G, K, dtype=torch.int32, device="cuda") for _ in range(3))
        assert lib.ncmb_beam_select(logits.data_ptr(), VOCAB, capi.F32, G, beams, VOCAB, scores.data_ptr(), done.data_ptr() if done is not None else None, EOS, K,
                                    *(t.data_ptr() for t in out)) == 0
        return out

    def reorder(self, parents):
        c, (t, n) = self.caches[self.at][0], ((self.table2, self.len2) if self.at == 0 else (self.table, self.len))
        assert lib.ncmb_paged_reorder(c, self.beams, parents.data_ptr(), LAYERS, self.pool.stride(1), t.data_ptr(), n.data_ptr(), None) == 0
        self.at ^= 1
        return n


def search(weights, prompts, beams, new, cache=torch.bfloat16):
    """(tokens [groups][beams][new], scores, done) of the best continuations, best first; prompts of one length."""
    G, n = len(prompts), len(prompts[0])
    m = Decoder(weights, G, beams, n, new, cache)
    ids = torch.tensor(prompts, device="cuda")
    for i in range(0, n, 128):                                    # the prompts, in pieces, into the groups' first rows
        piece = ids[:, i:i + 128]
        logits = m.forward(piece.reshape(-1), m.firsts, G).view(G, -1, VOCAB)[:, -1].contiguous()
        m.first_len += piece.shape[1]
    m.len[::beams] = n
    scores, parents, tokens, done = m.select(logits, 1, torch.zeros(G, 1, device="cuda"), None)
    lens = m.reorder(parents)                                     # all beams go on as row 0
    text = tokens[:, :, None]
    for _ in range(new - 1):
        logits = m.forward(tokens.view(-1).long(), m.caches[m.at], m.rows)
        lens += 1
        scores, parents, tokens, done = m.select(logits, beams, scores, done)
        lens = m.reorder(parents)
        text = torch.cat([text.gather(1, parents.long()[:, :, None].expand_as(text)), tokens[:, :, None]], 2)
    torch.cuda.synchronize()
    return text, scores, done


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--prompts", type=int, default=3)
    ap.add_argument("--beams", type=int, default=4)
    ap.add_argument("--new", type=int, default=24)
    ap.add_argument("--cache", choices=["f32", "bf16"], default="bf16")
    a = ap.parse_args()
    g = torch.Generator().manual_seed(1)
    prompts = torch.randint(0, VOCAB, (a.prompts, 200), generator=g).tolist()
    text, scores, done = search(Weights(0), prompts, a.beams, a.new, torch.float32 if a.cache == "f32" else torch.bfloat16)
    for g in range(a.prompts):
        for k in range(a.beams):
            print("prompt %d beam %d  %8.3f%s  %s" % (g, k, scores[g, k], " ended" if done[g, k] else "      ", text[g, k].tolist()))
