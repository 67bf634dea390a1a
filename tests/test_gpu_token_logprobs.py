"""Log probabilities of given tokens, their ranks, the entropy and the most probable tokens against the
definition in 64 bits.  Ranks and indices are exact; the others are within what the F32 steps can do,
derived in `bounds`."""
import numpy as np
import pytest
import torch

from gpu_util import announce, require_gpu

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module")
def S():
    require_gpu()
    import syntropy_amd.gemv as S
    return S


def exact(x, tokens, top, scale):
    """(logprob, rank, entropy, ids, top logprobs, and what the first, third and last may be off by)."""
    v = x.double().cpu().numpy()
    rows, vocab = v.shape
    with np.errstate(all="ignore"):
        z = v * scale
        m = z.max(1, keepdims=True)
        none = (m == -np.inf)[:, 0]
        d = np.where(none[:, None], -np.inf, z - m)
        p = np.exp(d)
        s = p.sum(1)
        p = p / s[:, None]
        lse = np.log(s)
        lp = d - lse[:, None]
        ent = -np.where(p > 0, p * lp, 0).sum(1)
    t = np.asarray(tokens.cpu())
    known = (t >= 0) & (t < vocab)
    at = np.where(known, t, 0)
    i = np.arange(rows)
    tlp = np.where(none, -np.inf, lp[i, at])
    ent = np.where(none, 0.0, ent)
    bad = np.isnan(z).any(1) | (z == np.inf).any(1)
    tlp, ent = np.where(bad, np.nan, tlp), np.where(bad, np.nan, ent)
    tlp = np.where(t < 0, 0.0, np.where(known, tlp, np.nan))
    rank = np.where(known, (v > v[i, at][:, None]).sum(1), -1)
    # greatest first, the lower index first among equals, a NaN before all (a stable sort puts them so)
    ids = torch.sort(x.double().cpu() + 0.0, dim=1, descending=True, stable=True).indices[:, :top].numpy()
    toplp = np.where(bad[:, None], np.nan, np.where(none[:, None], -np.inf, np.take_along_axis(lp, ids, 1)))
    # What the F32 steps move: x - m and its products by the scale and by log2(e) are rounded (3 U |d|), an
    # exponential is within 2 steps and follows its argument, a lane adds at most vocab / 64 terms in a chain and
    # the lanes' sums in 16 more; Z, U |z| twice, is room for the rescaling of a running sum.
    with np.errstate(all="ignore"):
        live = p > 0
        Z = np.where(live, np.abs(z), 0).max(1)
        D = np.where(live, p * np.abs(d), 0).sum(1)
        D2 = np.where(live, p * d * d, 0).sum(1)
        L = vocab / 64 + 16
        ds = U * (2 * Z + 2 * D + 4 + L)  # the sum's relative error, so log s's absolute one
        e_lp = 1.05 * (ds + U * (3 * np.abs(lse) + 2 * Z)) + 1e-30

        def off(l, dd):
            return np.where(np.isfinite(l), e_lp[:, None] + 1.05 * U * (2 * np.abs(dd) + 2 * np.abs(l)), 0)
        e_tok = off(lp, d)
        # e / s: each term's own error, its argument's, the chain's; then the quotient and the difference
        e_ent = 1.05 * (e_lp + U * (D * (2 * Z + 8 + L) + 2 * Z + 2 * D2 + 2 * D) + D * ds + U * np.abs(ent)) + 1e-30
    return (tlp, rank, ent, ids, toplp), (e_tok[i, at], e_ent, np.take_along_axis(e_tok, ids, 1))


def near(got, want, tol, what):
    got = got.double().cpu().numpy()
    assert got.shape == want.shape, what
    with np.errstate(invalid="ignore"):
        want = np.where(np.abs(want) >= 2.0 ** 128 * (1 - U / 2), np.sign(want) * np.inf, want)  # past F32's range
        ok = (np.abs(got - want) <= tol) | (got == want) | (np.isnan(got) & np.isnan(want))
    assert ok.all(), f"{what}: {int((~ok).sum())} of {ok.size}: {got[~ok][:3]} for {want[~ok][:3]} +- {np.asarray(tol)[~ok][:3]}"


def check(S, x, tokens, top, scale=1.0, what="", stream=None):
    announce(f"token_logprobs {tuple(x.shape)} {x.dtype} top {top} scale {scale} {what}")
    r = S.token_logprobs(x, tokens, top=top, scale=scale, stream=stream)
    torch.cuda.synchronize()
    (lp, rank, ent, ids, toplp), (e_lp, e_ent, e_top) = exact(x, tokens, top, float(np.float32(scale)))
    assert r.rank.dtype == torch.int32 and r.top_ids.dtype == torch.int32
    assert (r.rank.cpu().numpy() == rank).all(), f"{what}: ranks {r.rank} for {rank}"
    assert r.top_ids.shape == ids.shape and (r.top_ids.cpu().numpy() == ids).all(), f"{what}: indices"
    near(r.logprob, lp, e_lp, f"{what}: logprob")
    near(r.entropy, ent, e_ent, f"{what}: entropy")
    near(r.top_logprobs, toplp, e_top, f"{what}: top logprobs")
    return r


def logits(rows, vocab, dtype, seed, hidden=0.0):
    g = torch.Generator().manual_seed(seed)
    x = 3 * torch.randn(rows, vocab, generator=g)
    t = torch.randint(vocab, (rows,), generator=g)
    x[torch.arange(rows), t] += 6
    if hidden:
        hide = torch.rand(rows, vocab, generator=g) < hidden
        hide[torch.arange(rows), t] = False
        x[hide] = float("-inf")
    return x.to(dtype).cuda(), t.cuda()


SIZES = [(1, 1, 1), (1, 2, 2), (3, 7, 5), (1, 64, 64), (2, 65, 20), (5, 100, 64), (1, 1000, 0), (4, 1023, 1),
         (17, 4096, 5), (1, 8192, 20), (2, 8193, 33), (1, 32064, 20), (9, 50257, 64), (1, 128256, 8), (30, 32064, 64),
         (300, 2000, 3), (700, 515, 10), (2100, 129, 2), (64, 20011, 17), (130, 70001, 20)]


@pytest.mark.parametrize("scale", [2.0 ** -64, 2.0 ** -20, 2.0 ** 20, 2.0 ** 64])
def test_scales_at_their_ends(S, scale):
    x, t = logits(7, 3001, torch.float32, 5, 0.3)
    check(S, x, t, 9, scale, "scale")
    check(S, x * min(1 / scale, 2.0 ** 120), t, 9, scale, "scale, logits as far apart as before")


def test_a_distance_past_f32_counts_as_hidden(S):
    big = torch.finfo(torch.float32).max
    x = torch.tensor([[big, -big, 0.0], [big, -big, 0.0]], device="cuda")
    r = S.token_logprobs(x, torch.tensor([1, 0], device="cuda"), top=3, scale=2.0 ** -20)
    assert r.logprob.tolist() == [-float("inf"), 0.0] and r.rank.tolist() == [2, 0] and r.entropy.tolist() == [0.0, 0.0]
    assert r.top_ids.tolist() == [[0, 2, 1]] * 2 and r.top_logprobs[0].tolist() == [0.0, -big * 2.0 ** -20, -float("inf")]


@pytest.mark.parametrize("rows,vocab,top", SIZES)
def test_is_its_definition(S, rows, vocab, top):
    for i, (dt, scale) in enumerate(((torch.float32, 1.0), (torch.bfloat16, 0.7), (torch.float16, 1.3))):
        x, t = logits(rows, vocab, dt, rows + vocab + i)
        check(S, x, t if i else t.int(), top, scale, "random")


@pytest.mark.parametrize("hidden", [0.5, 0.95, 0.9999])
def test_hidden_tokens(S, hidden):
    for dt in (torch.float32, torch.bfloat16, torch.float16):
        for rows, vocab in ((1, 33000), (40, 3001), (600, 700)):
            x, t = logits(rows, vocab, dt, 5, hidden)
            check(S, x, t, 12, 1.0, f"hidden {hidden}")


@pytest.mark.parametrize("rows,vocab", [(14, 300), (14, 9000), (14, 70001), (560, 1500)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_rows_of_every_kind(S, rows, vocab, dtype):
    """Nothing visible, one visible, all equal, the type's lowest value as a mask, NaN, both infinities,
    zeros of both signs, ascending and descending values, large magnitudes."""
    x, t = logits(rows, vocab, torch.float32, 3)
    low = torch.finfo(dtype).min
    ramp = torch.arange(vocab, device="cuda", dtype=torch.float32) / vocab * 20
    for r in range(0, rows, 14):
        x[r] = float("-inf")
        x[r + 1] = float("-inf")
        x[r + 1, vocab - 1] = -3.0
        x[r + 2] = 1.5
        x[r + 3] = low
        x[r + 4, : vocab - 2] = low
        x[r + 5, vocab // 2] = float("nan")
        x[r + 6, 11] = float("inf")
        x[r + 7] = float("nan")
        x[r + 8] = torch.where(torch.arange(vocab, device="cuda") % 3 == 0, 0.0, -0.0)
        x[r + 9] = ramp
        x[r + 10] = -ramp
        x[r + 11] = 3e4 * torch.sin(torch.arange(vocab, device="cuda"))
        x[r + 12, ::2] = float("-inf")
        x[r + 13, 5] = float("inf")
        x[r + 13, 6] = float("-inf")
        x[r + 13, 250] = float("nan")
        t[r + 1] = vocab - 1
    t[0::14] = 0
    t[2::14] = vocab // 3
    x = x.to(dtype)
    for top, scale in ((0, 1.0), (5, 1.0), (64, 0.5), (20, 2.0)):
        check(S, x, t, top, scale, "every kind")


def test_tokens_that_are_none(S):
    """Negative: none asked for; vocab and more, past 32 bits too: none there."""
    x, t = logits(6, 500, torch.float32, 1)
    t[:] = torch.tensor([-1, 500, 3, -(1 << 40), 1 << 40, (1 << 32) + 3])
    check(S, x, t, 4, what="tokens")
    check(S, x, t[:3].int().repeat(2), 4, what="tokens")


def test_equal_values_go_by_index(S):
    """Few distinct values over a long row, so that equal ones fill the list and pass its end."""
    for vocab in (200, 5000, 128256):
        g = torch.Generator().manual_seed(vocab)
        x = torch.randint(0, 3, (3, vocab), generator=g).float()
        x[1] = (torch.arange(vocab) >= vocab - 70).float()   # the equal greatest ones at the end
        x[2] = (torch.arange(vocab) % 97 == 0).float()
        for top in (1, 7, 64):
            check(S, x.bfloat16().cuda(), torch.tensor([5, vocab - 1, 96]).cuda(), top, what="ties")


@pytest.mark.parametrize("rows,vocab", [(2, 700), (3, 40000), (1, 128256), (300, 900)])
def test_more_candidates_than_are_held_at_once(S, rows, vocab):
    """Rows whose greatest values rise along the row, or are as many as half of it, so that what passes the first
    bound is many times what is gathered at once; the same call gives the same bits."""
    i = torch.arange(vocab, device="cuda")
    for x in ((i // 8).float(), (i % 16 == 3).float(), (i % 2).float(), (i // 1024).float(), (vocab - i).float() // 100):
        x = (x * 2.0 ** -7).repeat(rows, 1)
        x[0, vocab // 2] = 5000.0
        t = torch.full((rows,), vocab - 1, device="cuda")
        r = check(S, x, t, 64, what="many candidates")
        for _ in range(3):
            again = S.token_logprobs(x, t, top=64)
            assert all(torch.equal(a, b) for a, b in zip(r, again))


def test_strided_unaligned_and_far_rows(S):
    x, t = logits(9, 3100, torch.float32, 2)
    for dt in (torch.float32, torch.bfloat16, torch.float16):
        y = x.to(dt)
        for first in (0, 1, 3):
            check(S, y[:, first:first + 3001], t % 3001, 9, what=f"from value {first}")
            check(S, y[:1, first:first + 3001], t[:1] % 3001, 9, what=f"from value {first}")
    far = 1 << 28  # rows more than 2^32 bytes from the first
    held = torch.empty(9 * far, dtype=torch.float32, device="cuda").as_strided((9, 3100), (far, 1))
    held.copy_(x)
    check(S, held, t, 9, what="far rows")


def test_a_row_does_not_depend_on_the_others(S):
    """However many rows are given, a row's indices, ranks and values agree within their roundings, and the
    same call gives the same bits."""
    x, t = logits(800, 6000, torch.bfloat16, 8)
    whole = S.token_logprobs(x, t, top=10)
    for rows in (1, 3, 40, 300):
        a, b = (S.token_logprobs(x[:rows], t[:rows], top=10) for _ in range(2))
        for u, v, w in zip(a, b, whole):
            assert torch.equal(u, v)
            if u.dtype == torch.int32:
                assert torch.equal(u, w[:rows])
        check(S, x[:rows], t[:rows], 10, what=f"{rows} rows")


def test_captured_and_replayed(S):
    for rows, vocab in ((1, 40000), (700, 900)):
        x, t = logits(rows, vocab, torch.float32, 1)
        S.token_logprobs(x, t, top=6)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        announce(f"capture {rows}x{vocab}")
        with torch.cuda.graph(graph):
            r = S.token_logprobs(x, t, top=6, scale=0.9)
        for i in range(3):
            y, u = logits(rows, vocab, torch.float32, 20 + i)
            x.copy_(y), t.copy_(u)
            want = S.token_logprobs(x, t, top=6, scale=0.9)
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(r, want):
                assert torch.equal(a, b)


def test_on_other_streams_at_once(S):
    sets = [logits(4, 50000, torch.float32, i) for i in range(2)]
    want = [S.token_logprobs(x, t, top=20) for x, t in sets]
    torch.cuda.synchronize()
    st = [torch.cuda.Stream(), torch.cuda.Stream()]
    announce("two streams")
    got = [[S.token_logprobs(x, t, top=20, stream=s if i else s.cuda_stream) for _ in range(5)]
           for i, ((x, t), s) in enumerate(zip(sets, st))]
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        for r in g:
            for a, b in zip(r, w):
                assert torch.equal(a, b)


def test_no_rows(S):
    r = S.token_logprobs(torch.empty(0, 50, device="cuda"), torch.empty(0, dtype=torch.int64, device="cuda"), top=3)
    assert r.logprob.shape == (0,) and r.top_ids.shape == (0, 3)


def test_a_feed_forward_block_and_head_to_the_next_token(S):
    """The operators together, as a serving step runs them: norm, gate/up, down, the residual, the head's
    logits, the log probabilities and the next token; captured, and against the same in 64 bits."""
    import syntropy_amd.int8 as I
    hidden, inter, vocab, rows = 512, 1400, 5003, 7
    g = torch.Generator().manual_seed(4)
    mats = [torch.randn(*s, generator=g) * 0.05 for s in ((2 * inter, hidden), (hidden, inter), (vocab, hidden))]
    gu, down, head = (I.quantize_weights(m.cuda()) for m in mats)
    gain = (torch.rand(hidden, generator=g) + 0.5).cuda()
    x = torch.randn(rows, hidden, generator=g).cuda()

    def step(x):
        h = I.gate_up_act(gu, S.rms_norm(x, gain, 1e-5, rows), rows)
        x = x + I.gemv(down, h, rows)
        lg = I.logits(head, gain, 1e-5, x, rows)
        first = S.token_logprobs(lg, torch.full((rows,), -1, device="cuda"), top=1)
        return lg, S.token_logprobs(lg, first.top_ids[:, 0].contiguous(), top=5)

    lg, r = step(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    announce("a step captured")
    with torch.cuda.graph(graph):
        held = step(x)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(held[0], lg) and all(torch.equal(a, b) for a, b in zip(held[1], r))
    assert (r.rank == 0).all()
    token = lg.argmax(1)
    (lp, rank, ent, ids, toplp), (e_lp, e_ent, e_top) = exact(lg, token, 5, 1.0)
    assert (r.top_ids.cpu().numpy() == ids).all()
    near(r.logprob, lp, e_lp, "logprob"), near(r.entropy, ent, e_ent, "entropy"), near(r.top_logprobs, toplp, e_top, "top")

    # in 64 bits, the rows quantized by the same rule: a code may move where a last bit moves it, each by one
    # step of its row, 1 / 127 of the largest value; over k of them that is a random walk of relative size
    # below 1e-3 of an output here, and far below that in the log probabilities
    def q64(v):
        s = v.abs().amax(1, keepdim=True) / 127
        return torch.round(v / s) * s

    def w64(w):
        return w.codes.double() * w.scales.double()[:, None]

    def norm(v):
        return v / torch.sqrt((v * v).mean(1, keepdim=True) + 1e-5) * gain.double()
    v = x.double()
    y = q64(norm(v)) @ w64(gu).t()
    y = torch.nn.functional.silu(y[:, :inter]) * y[:, inter:]
    v = v + q64(y) @ w64(down).t()
    want = q64(norm(v)) @ w64(head).t()
    assert ((lg.double() - want).norm() / want.norm()) < 1e-2
