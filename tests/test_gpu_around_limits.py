"""Dropout, the scaled lookup and group norm at the ends of what they take: the largest values and sizes, the longest sums, sums that are exact."""
import pytest
import torch

import test_gpu_norm as norm_checks
from dfa3D.dropout import dropout
from dfa3D.embedding import scaled_embedding
from dfa3D.norm import level_group_norm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,S,C,G,start", [(6, 4001, 256, 32, (0, 3015, 3797)), (1, 40000, 16, 2, (0, 39999)), (2, 30001, 48, 3, None)])
def test_norm_of_values_whose_squares_are_too_large(B, S, C, G, start, dtype):
    """Values of some 3e19, whose squares leave the type that sums are formed in, all close together: their mean's error counts, e = 80 u 3e19 = 1.5e14 for a
    deviation of 2e17, and nothing is infinite.  Levels that have fewer keys in a tile than the threads side by side: some of those have none."""
    torch.manual_seed(S)
    step = 2.0 ** 57                                             # of bfloat16 from 2^64 to 2^65
    x = (2.0 ** 64 * 1.5 + step * torch.randint(-2, 3, (B, S, C), device="cuda")).to(dtype)
    assert bool(x.isfinite().all()) and bool((x.double() >= 2.0 ** 64).all())
    norm_checks.check(x, G, *norm_checks.params(C, dtype), start=start, act="silu")


def whole_sums(R, N, V, H, E, dtype, scaled, index, seed=0):
    """The gradients of a table and of its scales where every sum is one of whole numbers below 2^24, which float holds exactly whatever the order: what is lost or
    counted twice shows, and only the last rounding to bfloat16 is left."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    whole = lambda low, high, *shape: torch.randint(low, high + 1, shape, generator=g, device="cuda")
    lead = () if R is None else (R,)
    table = whole(-3, 3, *((V, H, E) if H else (V, E))).to(dtype).requires_grad_()
    wide = torch.float64 if dtype == torch.float64 else torch.float32
    scale = whole(1, 2, *lead, N, *((H,) if H else ())).to(wide).requires_grad_() if scaled else None
    plus = torch.zeros(*lead, N, E, dtype=dtype, device="cuda") if lead and not scaled else None
    grad = whole(-2, 4, *lead, N, E).to(dtype)
    out = scaled_embedding(table, index, scale=scale, plus=plus)
    got = torch.autograd.grad(out, (table, scale) if scaled else table, grad)
    there = (index >= 0) & (index < V)
    at = index.long()[there]
    rows = grad.reshape(-1, N, E)[:, there]
    want = torch.zeros(V, max(H, 1), E, dtype=torch.int64, device="cuda")
    by = None if scale is None else scale.detach().reshape(len(rows), N, max(H, 1))[:, there].long()
    for r0 in range(0, len(rows), 64):
        piece = rows[r0:r0 + 64].long()[:, :, None, :].expand(-1, -1, max(H, 1), -1)
        want.index_add_(0, at, (piece if by is None else piece * by[r0:r0 + 64, :, :, None]).sum(0))
    assert int(want.abs().max()) < 2 ** 24
    assert torch.equal(got[0], want.view(table.shape).double().to(dtype))
    if scaled:
        dots = torch.zeros(len(grad.reshape(-1, N, E)), N, max(H, 1), dtype=torch.int64, device="cuda")
        dots[:, there] = (rows.long()[:, :, None, :] * table.detach().reshape(V, max(H, 1), E)[at].long()[None]).sum(-1)
        assert torch.equal(got[1], dots.view(scale.shape).to(wide))


@pytest.mark.parametrize("dtype,scaled", [(torch.float32, True), (torch.bfloat16, False)])
@pytest.mark.parametrize("R,N,V,H,E", [(10000, 100, 100, 0, 64), (20000, 100, 100, 0, 64), (20000, 60, 100, 2, 12), (3000, 700, 131073, 0, 8), (64, 20000, 100, 0, 256), (9, 120000, 50, 3, 16)])
def test_lookup_of_many_batch_elements(R, N, V, H, E, dtype, scaled):
    """On both sides of 2^20 places of all batch elements, and of the rule by which those are places of their own."""
    index = torch.randint(-1, V + 1, (N,), generator=torch.Generator().manual_seed(R)).cuda()
    index[N // 2] = V - 1
    whole_sums(R, N, V, H, E, dtype, scaled, index)


def test_lookup_of_more_batch_elements_than_float_counts():
    """One place of 2^25 batch elements whose gradients are ones: a float that adds them up one after the other stops at 2^24."""
    R = 2 ** 25
    for scaled in (False, True):
        table = torch.randn(3, 4, device="cuda", requires_grad=True)
        ones = torch.ones(R, 1, device="cuda") if scaled else None
        out = scaled_embedding(table, torch.tensor([1], device="cuda"), scale=ones, plus=None if scaled else torch.zeros(R, 1, 4, device="cuda"))
        grad, = torch.autograd.grad(out, table, torch.ones_like(out))
        assert torch.equal(grad, torch.tensor([0.0, R, 0.0], device="cuda")[:, None].expand(3, 4))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,S,start", [(17000000, 1, None), (2 ** 24 - 1, 1, None), (8400001, 2, (0, 1))])
def test_norm_of_more_batch_elements_than_a_grid_holds(B, S, start, dtype):
    """Tiles of all batch elements in turns."""
    torch.manual_seed(S)
    x = torch.empty(B, S, 8, device="cuda", dtype=dtype).normal_()
    norm_checks.check(x, 2, *norm_checks.params(8, dtype), start=start)
    torch.cuda.empty_cache()


def _one_entry(N, V):
    index = torch.randint(0, V, (N,))
    index[N // 3:N // 2], index[N // 2:N // 2 + 40] = V - 1, V // 2
    outside = torch.rand(N) < 0.2
    index[outside] = torch.tensor([-1, V, -V - 5, 2 ** 31 - 1])[torch.randint(0, 4, (int(outside.sum()),))]
    return index


def _low_entries(N, V):
    return ((torch.rand(N, dtype=torch.float64) * 11.0).exp() - 1).long().clamp(max=V - 1)


def _long_runs(N, V):
    index = torch.randint(0, V, (N,))
    index[N // 4:N // 2], index[N // 2:N // 2 + 17], index[-700:] = V - 1, 7, min(V - 1, 262144)
    return index


@pytest.mark.parametrize("index_type", [torch.int32, torch.int64])
@pytest.mark.parametrize("made,N,V", [(_one_entry, 65536, 131072), (_one_entry, 65537, 1), (_one_entry, 70001, 1024), (_one_entry, 100003, 2 ** 20 + 1), (_one_entry, 131071, 3),
                                      (_one_entry, 70000, 2 ** 22 + 2047), (_low_entries, 60000, 90000), (_low_entries, 90000, 60000), (_long_runs, 20011, 400001), (_long_runs, 30000, 50),
                                      (_long_runs, 1048576, 500), (_low_entries, 1048577, 50000)])
def test_lookup_sums_of_whole_numbers(made, N, V, index_type):
    """Entries of very many places, whose sums are cut in pieces, in both ways of ordering: no place is lost or counted twice."""
    torch.manual_seed(N + V)
    index = made(N, V).to(index_type).cuda()
    whole_sums(None, N, V, 0, 6, torch.float32, True, index)
    whole_sums(2, N, V, 2, 4, torch.float32, True, index)
    whole_sums(None, N, V, 5, 8, torch.bfloat16, True, index)
    whole_sums(None, N, V, 0, 40, torch.bfloat16, False, index)


@pytest.mark.parametrize("act", [None, "silu"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("S,C", [(127, 513), (64, 1023), (90, 721)])
def test_norm_of_the_longest_sums_in_a_thread(S, C, dtype, act):
    """One launch, one key at a time beside 513 to 1024 pieces of one channel: a thread adds up as many terms of a channel as there are keys, up to 127 (2^16 elements of
    a group in 513 pieces), before anything is in double.  Bounds as in the tests of the norm, whose 80 u for sums are 136 u here: at most 1.7 times them."""
    torch.manual_seed(S)
    x = (torch.randn(1, S, C, device="cuda") + torch.randn(C, device="cuda")).to(dtype).requires_grad_()
    w, b = (t.requires_grad_() for t in norm_checks.params(C, dtype))
    y = level_group_norm(x, 1, w, b, act=act)
    g = torch.randint(-4, 5, y.shape, device="cuda").to(dtype)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), g)
    with torch.no_grad():
        want = norm_checks.formulas(x, 1, w, b, None, 1e-5, act, g, dtype)
    for got, (value, off), kind, name in ((y, want[0], dtype, "y"), (dx, want[1], dtype, "dx"), (dw, want[2], torch.float32, "dw"), (db, want[3], torch.float32, "db")):
        norm_checks.close(got, value, 1.7 * off, kind, name)
    if act is None:
        assert torch.equal(db, g.double().sum((0, 1)).float())   # whole numbers: exact


def test_dropout_draws_the_published_words():
    """Philox4x32 of seven rounds at a counter and a key of zero, from the authors' table of known answers: an element is kept where p 2^32 is its word, and dropped where it
    is one more."""
    x = torch.ones(4, device="cuda")
    for k, word in enumerate((0x5F6FB709, 0x0D893F64, 0x4F121F81, 0x4F730A48)):
        assert dropout(x, word / 2.0 ** 32, 0, 0)[k] > 0 and dropout(x, (word + 1) / 2.0 ** 32, 0, 0)[k] == 0
