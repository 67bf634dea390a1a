"""Sampling against its definition in 64 bits.  Tokens and counts are equal; a log probability is F32's nearest to
within the 64-bit steps."""
import numpy as np
import pytest
import torch

from gpu_util import announce, require_gpu

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def S():
    require_gpu()
    import syntropy_amd.gemv as S
    return S


def real(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def uniform(seed, *shape):
    return torch.rand(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def f32(v):
    return float(np.float32(v))


def one(z, u, temperature, top_k, top_p, min_p):
    """(token, logprob, kept, how near the nearest border is) of one row, z in 64 bits."""
    order = np.argsort(-z, kind="stable")
    z = z[order]
    n = int((z > -np.inf).sum())
    if temperature == 0:
        temperature, top_k = 1.0, 1
    if 0 < top_k < n:
        n = int(top_k)
    w = np.exp((z[:n] - z[0]) / temperature)
    run, gap = np.cumsum(w), 1.0
    if top_p < 1:
        gap = min(gap, np.abs(run / run[-1] - top_p).min())
        n = min(n, 1 + int((run < top_p * run[-1]).sum()))
    if min_p > 0:
        gap = min(gap, np.abs(w - min_p)[w < 1].min(initial=1.0))  # (a weight of 1 is exact)
        n = min(n, int((w >= min(min_p, 1.0)).sum()))
    run = run[:n]
    gap = min(gap, np.abs(run / run[-1] - u).min())
    at = min(int((run <= u * run[-1]).sum()), n - 1)
    return int(order[at]), np.log(w[at] / run[-1]), n, gap


def check(S, x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, near=1e-11, what="", ends=0):
    """ends: rows whose u is the greatest.  What is behind it, 2^-24 of the sum, may be thousands of values of less than
    `near` each: such a row's token is one whose share of [0, 1) reaches to within `near` of u."""
    r = S.sample_tokens(x, u, temperature, top_k, top_p, min_p)
    rows = x.shape[0]
    z, us = x.double().cpu().numpy(), u.double().cpu().numpy()
    got = [t.cpu().numpy() for t in r]
    assert got[0].dtype == np.int32 and got[1].dtype == np.float32 and got[2].dtype == np.int32

    def at(v, i):
        return float(v[i]) if torch.is_tensor(v) else f32(v)
    skipped = 0
    for i in range(rows):
        tok, lp, n, gap = one(z[i], us[i], at(temperature, i), at(top_k, i), at(top_p, i), at(min_p, i))
        if gap < near:  # (the 64-bit sums of the test are not exact either)
            skipped += 1
            if ends and us[i] == 1 - 2.0 ** -24:
                order = np.argsort(-z[i], kind="stable")[:got[2][i]]
                run = np.cumsum(np.exp((z[i][order] - z[i][order[0]]) / at(temperature, i)))
                place = int(np.nonzero(order == got[0][i])[0][0])
                assert run[place] / run[-1] > us[i] - near and (run[place - 1] if place else 0.0) / run[-1] < us[i] + near
            continue
        assert (got[0][i], got[2][i]) == (tok, n), f"{what} row {i}: token {got[0][i]}, kept {got[2][i]}, not {tok}, {n}"
        assert abs(got[1][i] - lp) <= 2.0 ** -24 * abs(lp) + 1e-9, f"{what} row {i}: logprob {got[1][i]}, not {lp}"
    assert skipped <= rows // 20 + ends, f"{skipped} rows next to a border"


FILTERS = [dict(), dict(top_k=1), dict(top_k=7), dict(top_k=300), dict(top_p=0.9), dict(top_p=0.01), dict(top_p=0.9999), dict(min_p=0.1),
           dict(min_p=1.0), dict(min_p=1e-6), dict(top_k=50, top_p=0.8), dict(top_k=1000, top_p=0.97, min_p=0.01, temperature=0.7),
           dict(temperature=0.0), dict(temperature=0.05), dict(temperature=9.0, top_p=0.5), dict(temperature=2.0, min_p=0.3, top_p=0.99)]


@pytest.mark.parametrize("ty", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [1, 2, 63, 64, 65, 1000, 1024, 1025, 5003, 32064, 50257])
def test_filters(S, vocab, ty):
    rows = 6 if vocab < 30000 else 3
    x = (3 * real(vocab, rows, vocab)).to(ty)
    for i, kw in enumerate(FILTERS):
        announce(f"sample {vocab} {ty} {kw}")
        # F16 and BF16 rows are full of equal logits; a min-p on one of their weights is a border (none here is)
        check(S, x, uniform(100 + i, rows), what=f"{kw}", **kw)


@pytest.mark.parametrize("rows,vocab", [(1, 128256), (2, 128256), (24, 128256), (100, 50257), (300, 8000), (700, 1111)])
def test_many_rows_and_wide_ones(S, rows, vocab):
    x = 2 * real(rows, rows, vocab)
    x.scatter_(1, torch.randint(vocab, (rows, 8), device="cuda"), 11 + 2 * real(rows + 1, rows, 8))
    for i, kw in enumerate((dict(), dict(top_k=40, top_p=0.95, temperature=0.8), dict(top_p=0.9), dict(min_p=0.05))):
        announce(f"sample {rows} {vocab} {kw}")
        check(S, x, uniform(i, rows), what=f"{kw}", **kw)


@pytest.mark.parametrize("ty", [F32, BF16], ids=["f32", "bf16"])
def test_each_row_its_own(S, ty):
    rows, vocab = 64, 5000
    x = (2.5 * real(1, rows, vocab)).to(ty)
    x[3], x[4] = -float("inf"), 0.5
    x[3, 77] = -3.0  # one visible logit; all equal
    t = 0.3 + 2 * uniform(2, rows)
    t[::7] = 0.0
    k = torch.randint(-2, 90, (rows,), dtype=torch.int32, device="cuda")
    k[4] = 0
    p = 0.3 + uniform(3, rows)
    mp = torch.where(uniform(4, rows) < 0.5, 0.0, 0.2 * uniform(5, rows))
    check(S, x, uniform(6, rows), t, k, p, mp)


def test_equal_logits_go_by_index(S):
    """All equal: token floor(u n), the first n = ceil(p vocab) kept; runs of equal ones at a cut."""
    for ty in (F32, F16, BF16):
        for vocab in (64, 1000, 40000):
            x = torch.full((5, vocab), -2.5, dtype=ty, device="cuda")
            u = torch.tensor([0.0, 0.25, 0.4999, 0.75, 1 - 2.0 ** -24], device="cuda")
            r = S.sample_tokens(x, u)
            assert r.token.tolist() == [int(v * vocab) for v in u.double().tolist()] and r.kept.tolist() == [vocab] * 5
            assert torch.allclose(r.logprob.cpu().double(), torch.full((5,), -np.log(vocab), dtype=torch.double), rtol=2.0 ** -24, atol=1e-9)
            r = S.sample_tokens(x, u, top_p=0.5)
            assert r.kept.tolist() == [vocab // 2] * 5 and r.token.tolist() == [int(v * (vocab // 2)) for v in u.double().tolist()]
            r = S.sample_tokens(x, u, top_k=7)
            assert r.kept.tolist() == [7] * 5 and r.token.tolist() == [int(v * 7) for v in u.double().tolist()]
            # +0 and -0 are equal
            z = torch.where(torch.arange(vocab, device="cuda") % 2 == 0, 0.0, -0.0).to(ty).repeat(5, 1)
            assert S.sample_tokens(z, u).token.tolist() == [int(v * vocab) for v in u.double().tolist()]


def test_next_to_every_border(S):
    """u the F32 number right below and right above where the running sum stands (not the nearest, which may be on
    either side of it): both neighbours of every border are found."""
    vocab = 600
    z = 1.5 * real(9, vocab)
    w = np.sort(np.exp(z.double().cpu().numpy()))[::-1]
    run = np.cumsum(w) / w.sum()
    edge = run[:-1].astype(np.float32)
    lo = np.nextafter(edge, np.float32(0))
    hi = np.nextafter(edge, np.float32(1))
    us = torch.from_numpy(np.concatenate([lo, hi])).cuda()
    check(S, z.repeat(len(us), 1), us, what="borders")


def test_hidden_logits(S):
    rows, vocab = 40, 20011
    x = 2 * real(1, rows, vocab)
    x[uniform(2, rows, vocab) < 0.97] = -float("inf")
    x[0] = -float("inf")
    x[0, vocab - 1] = -1e30
    x[1] = -float("inf")
    x[1, [5, 900]] = torch.tensor([3e38, -3e38], device="cuda")
    for kw in (dict(), dict(top_k=2000), dict(top_p=0.7), dict(min_p=0.01), dict(top_k=2)):
        check(S, x, uniform(3, rows), what=f"{kw}", **kw)


def test_type_lowest_values_as_a_mask(S):
    """A mask of the type's lowest value hides nothing: such logits count, with a weight of nothing."""
    for ty in (F32, F16, BF16):
        x = (2 * real(1, 8, 3000)).to(ty)
        x[:, ::2] = torch.finfo(ty).min
        for kw in (dict(), dict(top_k=2900), dict(top_p=0.99), dict(min_p=1e-9)):
            check(S, x, uniform(2, 8), what=f"{ty} {kw}", **kw)


def test_rows_without_a_distribution(S):
    x = real(1, 8, 700)
    x[0] = -float("inf")
    x[1, 699] = float("nan")
    x[2, 0] = float("inf")
    t = torch.ones(8, device="cuda")
    t[3], t[4] = float("nan"), -1.0
    p = torch.ones(8, device="cuda")
    p[5] = float("nan")
    u = torch.full((8,), 0.5, device="cuda")
    u[6] = float("nan")
    r = S.sample_tokens(x, u, temperature=t, top_p=p)
    assert r.token[:7].tolist() == [-1] * 7 and r.kept[:7].tolist() == [0] * 7 and bool(torch.isnan(r.logprob[:7]).all())
    assert int(r.token[7]) >= 0 and int(r.kept[7]) == 700


def test_settings_and_u_outside_their_ranges(S):
    x, n = real(1, 6, 500), 500
    full = torch.full
    u = torch.tensor([-0.5, 1.0, 2.0, -float("inf"), float("inf"), 0.3], device="cuda")
    lo, hi = torch.zeros(6, device="cuda"), full((6,), 1 - 2.0 ** -24, device="cuda")
    r, a, b = S.sample_tokens(x, u), S.sample_tokens(x, lo), S.sample_tokens(x, hi)
    assert r.token[[0, 3]].tolist() == a.token[[0, 3]].tolist() and r.token[[1, 2, 4]].tolist() == b.token[[1, 2, 4]].tolist()
    u = uniform(5, 6)
    assert S.sample_tokens(x, u, top_p=full((6,), -1.0, device="cuda")).kept.tolist() == [1] * 6
    assert S.sample_tokens(x, u, top_p=full((6,), 7.0, device="cuda")).kept.tolist() == [n] * 6
    assert S.sample_tokens(x, u, min_p=full((6,), 3.0, device="cuda")).kept.tolist() == [1] * 6
    assert S.sample_tokens(x, u, min_p=full((6,), -3.0, device="cuda")).kept.tolist() == [n] * 6
    assert S.sample_tokens(x, u, top_k=full((6,), -3, dtype=torch.int32, device="cuda")).kept.tolist() == [n] * 6
    assert S.sample_tokens(x, u, top_k=10 ** 6).kept.tolist() == [n] * 6


def test_strided_rows_streams_and_graphs(S):
    wide = torch.full((9, 4013), float("nan"), device="cuda")
    x = wide[:, 3:4003]
    x.copy_(2 * real(1, 9, 4000))
    u = uniform(2, 9)
    check(S, x, u, top_p=0.9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    r = S.sample_tokens(x, u, top_p=0.9, stream=side)
    side.synchronize()
    want = S.sample_tokens(x.contiguous(), u, top_p=0.9)
    assert all(torch.equal(a, b) for a, b in zip(r, want))
    t = torch.full((9,), 0.7, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r = S.sample_tokens(x, u, temperature=t, top_k=30)
    for i in range(4):
        u.copy_(uniform(10 + i, 9))
        t.fill_(0.5 + 0.2 * i)
        x.copy_(2 * real(30 + i, 9, 4000))
        g.replay()
        got = [v.clone() for v in r]
        torch.cuda.synchronize()
        want = S.sample_tokens(x, u, temperature=t, top_k=30)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


def test_no_rows(S):
    r = S.sample_tokens(torch.zeros(0, 50, device="cuda"), torch.zeros(0, device="cuda"))
    assert [t.shape for t in r] == [(0,)] * 3


def spread(rows):
    """How often rows are repeated to be more than are shared out between workgroups."""
    return -(-200 // rows)


@pytest.mark.parametrize("ty", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("temperature", [0.5, 1.4, 3.0, 5.0, 30.0])
def test_flat_rows(S, ty, temperature):
    """Bins of hundreds and of thousands of values: border and token in one list, in two, and past a list."""
    rows, vocab = 6, 128256
    x = (2 * real(7, rows, vocab)).to(ty)
    u = uniform(8, rows)
    u[0], u[1] = 0.0, 1 - 2.0 ** -24
    for kw in (dict(), dict(top_p=0.93), dict(top_p=0.4), dict(min_p=0.2), dict(top_p=0.8, min_p=0.05), dict(top_p=0.6, top_k=60000)):
        announce(f"sample flat {ty} {temperature} {kw}")
        check(S, x, u, temperature, what=f"{kw}", ends=1, **kw)
        n = spread(rows)
        few, many = S.sample_tokens(x, u, temperature, **kw), S.sample_tokens(x.repeat(n, 1), u.repeat(n), temperature, **kw)
        for a, b in zip(few, many):
            assert torch.equal(a.repeat(n), b), kw


@pytest.mark.parametrize("ty", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab", [(4, 9000), (4, 131071), (130, 70001)])
def test_most_of_a_row_far_below(S, rows, vocab, ty):
    """Weights below 2^-64 beside a few that count: they are counted, and never the token."""
    x = real(3, rows, vocab) - 300
    x.scatter_(1, torch.randint(vocab, (rows, 150), generator=torch.Generator(device="cuda").manual_seed(4), device="cuda"),
               2 * real(5, rows, 150))
    x = x.to(ty)
    u = uniform(6, rows)
    u[0], u[-1] = 1 - 2.0 ** -24, 0.0
    for kw in (dict(), dict(top_k=400), dict(top_k=60), dict(top_k=5000), dict(top_p=0.99), dict(min_p=1e-4), dict(top_p=0.5, min_p=0.3)):
        announce(f"sample far {rows} {vocab} {ty} {kw}")
        check(S, x[:4], u[:4], what=f"{kw}", ends=1, **kw)
        many, few = S.sample_tokens(x, u, **kw), S.sample_tokens(x[:4], u[:4], **kw)
        assert all(torch.equal(a[:4], b) for a, b in zip(many, few))


@pytest.mark.parametrize("ty", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
def test_long_rows_shared_by_workgroups(S, ty):
    """Each way to a row's list, in rows that several workgroups read, each row with its own settings."""
    rows, vocab = 14, 100003
    x = 2 * real(11, rows, vocab)
    x.scatter_(1, torch.randint(vocab, (rows, 9), generator=torch.Generator(device="cuda").manual_seed(12), device="cuda"),
               11 + 2 * real(13, rows, 9))
    x[5:7] = x[5:7].bfloat16().float()
    x = x.to(ty)
    none = torch.tensor([0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 1, 1, 1], dtype=torch.bool)
    x[11], x[12, 99999], x[13, 7] = -float("inf"), float("nan"), float("inf")
    t = torch.tensor([1, .7, 0, 1.2, .9, 1, 1.1, 2, .5, 1, .8, 1, 1, 1], device="cuda")
    k = torch.tensor([0, 7, 0, 64, 65, 700, 1984, 1985, 30000, 0, 0, 3, 0, 900], dtype=torch.int32, device="cuda")
    p = torch.tensor([1, .9, 1, 1, .95, 1, .99, .8, .9, .9, 1, .9, 1, 1], device="cuda")
    mp = torch.tensor([0, 0, 0, 0, .001, 0, 0, 0, .0001, .01, .02, 0, 0, .1], device="cuda")
    for seed in range(3):
        u = uniform(20 + seed, rows)
        check(S, x[:11], u[:11], t[:11], k[:11], p[:11], mp[:11])
        r = S.sample_tokens(x, u, t, k, p, mp)
        assert r.token.cpu()[none].tolist() == [-1] * 3 and r.kept.cpu()[none].tolist() == [0] * 3
        assert bool(torch.isnan(r.logprob.cpu()[none]).all())
        n = spread(rows)
        many = S.sample_tokens(x.repeat(n, 1), u.repeat(n), t.repeat(n), k.repeat(n), p.repeat(n), mp.repeat(n))
        for a, b in zip(r, many):
            assert torch.equal(torch.nan_to_num(a.float(), -9.0).repeat(n), torch.nan_to_num(b.float(), -9.0))


def test_two_calls_at_once(S):
    """On two streams, each with its own workspace, and a call that is replayed between them."""
    xs, us = [2 * real(i, 5, 128256) for i in range(3)], [uniform(9 + i, 5) for i in range(3)]
    want = [S.sample_tokens(x, u, top_p=0.95) for x, u in zip(xs, us)]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kept = S.sample_tokens(xs[2], us[2], top_p=0.95)
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in sides:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(6):
        for i, s in enumerate(sides):
            got[i].append(S.sample_tokens(xs[i], us[i], top_p=0.95, stream=s))
        g.replay()
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(r, want[i]))
    assert all(torch.equal(a, b) for a, b in zip(kept, want[2]))
