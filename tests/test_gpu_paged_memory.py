"""Arrays side by side, with nothing between them, and results in place where that is allowed: taken."""
import pytest
import torch

import helpers

pytestmark = pytest.mark.gpu
capi = helpers.capi


def test_side_by_side():
    cuda = capi.NcmLib(helpers.CUDA_LIB)
    G, K, V = 3, 4, 1000
    for n in (4, 7):
        words = torch.zeros(G * K * (V + 2) + 4 * G * n, device="cuda")
        x, scores, done = words[:G * K * V], words[G * K * V:G * K * (V + 1)], words[G * K * (V + 1):G * K * (V + 2)]
        x.copy_(torch.randn(G * K * V, device="cuda"))
        scores.copy_(-torch.rand(G * K, device="cuda"))
        out = [words[G * K * (V + 2) + i * G * n:][:G * n] for i in range(4)]
        args = (x.data_ptr(), V, capi.F32, G, K, V, scores.data_ptr(), done.data_ptr(), 3, n)
        assert cuda.ncmb_beam_select(*args, *(o.data_ptr() for o in out)) == 0
        torch.cuda.synchronize()
        assert (out[0].view(G, n)[:, :-1] >= out[0].view(G, n)[:, 1:]).all() and out[0].max() < 0
        if n == K:                                              # in place
            want = [o.clone() for o in out]
            assert cuda.ncmb_beam_select(*args, scores.data_ptr(), out[1].data_ptr(), out[2].data_ptr(), done.data_ptr()) == 0
            torch.cuda.synchronize()
            assert torch.equal(scores, want[0]) and torch.equal(out[1].view(torch.int32), want[1].view(torch.int32)) and torch.equal(done.view(torch.int32), want[3].view(torch.int32))
    rows, width, pages = 6, 4, 24
    k = torch.randn(pages, 1, 8, 8, device="cuda")
    ints = torch.zeros(2 * rows * width + 3 * rows + pages, dtype=torch.int32, device="cuda")
    at, parts = 0, []
    for n in (rows * width, rows, rows, rows * width, rows, pages):
        parts.append(ints[at:at + n])
        at += n
    table, lens, parents, t2, l2, refs = parts
    table.copy_(torch.arange(pages, device="cuda"))
    lens.fill_(3)
    parents.copy_(torch.tensor([1, 1, 0, 2, 2, 2], device="cuda"))
    c = capi.PagedCache.of(k, k.clone(), table.view(rows, width), lens)
    assert cuda.ncmb_paged_reorder(c, 3, parents.data_ptr(), 1, 0, t2.data_ptr(), l2.data_ptr(), refs.data_ptr()) == 0
    torch.cuda.synchronize()
    assert t2.view(rows, width)[:, 0].tolist() == [4, 8, 0, 20, 12, 16] and (l2 == 3).all() and (refs == 0).all()
