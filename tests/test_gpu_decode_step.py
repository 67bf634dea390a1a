"""The operators of a step together, as a model's loop calls them: norms between blocks, a gated feed-forward block,
logits, a token; eager and as one captured graph."""
import pytest
import torch

from gpu_util import require_gpu

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
HID, INTER, VOCAB, LAYERS, EPS = 512, 1408, 3001, 2, 1e-5


def real(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


@pytest.mark.parametrize("rows", [1, 5, 40])
def test_a_step(rows):
    require_gpu()
    import syntropy_amd.gemv as S
    import syntropy_amd.half as H
    import syntropy_amd.int8 as I

    def weights(seed, n, k):
        return H.Weights((real(seed, n, k) / k ** 0.5).to(BF16))
    layers = [dict(mix=weights(10 * i + 1, HID, HID), up=weights(10 * i + 2, INTER, HID), gate=weights(10 * i + 3, INTER, HID),
                   down=weights(10 * i + 4, HID, INTER), g1=1 + 0.1 * real(10 * i + 5, HID), g2=1 + 0.1 * real(10 * i + 6, HID),
                   post=1 + 0.1 * real(10 * i + 7, HID)) for i in range(LAYERS)]
    head, gain = I.quantize_weights(real(90, VOCAB, HID) / HID ** 0.5 * 4), 1 + 0.1 * real(91, HID)
    x, u = real(92, rows, HID).to(BF16), torch.rand(rows, device="cuda")

    def step():
        h, b = x, None
        for l in layers:
            h, y = S.block_norm(h, b, l["g1"], EPS, rows)
            h, y = S.block_norm(h, H.gemv(l["mix"], y, rows), l["g2"], EPS, rows, post=l["post"])
            up = H.gemv(l["up"], y, rows)
            b = H.gemv(l["down"], H.gemv(l["gate"], y, rows, act="silu", gate=up), rows)
        h, _ = S.block_norm(h, b, None, EPS, rows)
        logits = I.logits(head, gain, EPS, h.float(), rows)
        return h, logits, S.sample_tokens(logits, u, temperature=0.8, top_k=50, top_p=0.9)

    def rms(v, g):
        return v / torch.sqrt((v * v).mean(1, keepdim=True) + EPS) * g.double()
    h, b = x.double(), torch.zeros(rows, HID, dtype=torch.double, device="cuda")
    for l in layers:
        h = h + b
        mixed = rms(h, l["g1"]) @ l["mix"].matrix.double().T
        h = h + rms(mixed, l["post"])
        y = rms(h, l["g2"])
        b = (torch.nn.functional.silu(y @ l["gate"].matrix.double().T) * (y @ l["up"].matrix.double().T)) @ l["down"].matrix.double().T
    h = h + b
    got, logits, r = step()
    # a stream of BF16 is rounded 5 times, each block's inputs, inner rows and output once: some 30 steps of 2^-9 of values
    # of at most 5 times the typical, in quadrature and in the worst case not
    assert float((got.double() - h).abs().max()) < 30 * 2.0 ** -9 * float(h.abs().max())
    # the token and its log probability are those of these logits
    z = logits.double() / float(torch.tensor(0.8))
    p = torch.softmax(z.gather(1, z.topk(50, 1).indices), 1)
    kept = 1 + (p.cumsum(1) < float(torch.tensor(0.9))).sum(1)
    assert torch.equal(kept.to(torch.int32), r.kept)
    lp = S.token_logprobs(logits, r.token, scale=1.25)
    # of all tokens, and of the kept ones: their difference is the kept ones' share
    share = torch.stack([torch.logsumexp(z[i].topk(int(k)).values, 0) - torch.logsumexp(z[i], 0) for i, k in enumerate(kept)])
    assert torch.allclose(lp.logprob.double() - share, r.logprob.double(), atol=1e-4)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for i in range(4):
        u.copy_(torch.rand(rows, device="cuda"))
        x.copy_(real(200 + i, rows, HID))
        g.replay()
        seen = [out[0].clone(), out[1].clone(), *(t.clone() for t in out[2])]
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(seen, [want[0], want[1], *want[2]])), i
