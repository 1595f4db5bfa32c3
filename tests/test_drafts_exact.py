"""Sampled decoding at its limits: verdicts that the caches' acceptance follows."""
import math

import pytest
import torch

from tests import gen
from tests.test_drafts import PROMPT, T, bit_words, host, small_model

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------
# acceptance
# ---------------------------------------------------------------------------

def caches_of(iw, B, N):
    """A chain's K and V with their caches, one layer of two heads."""
    r = gen.rng(B + N)
    qkv = T(gen.i8(r, (B, N, 3 * 128)))
    k, v = (torch.zeros(s, dtype=torch.int8, device="cuda") for s in ((B, 2, 64, 64), (B, 2, 16, 64, 4)))
    return iw.speculative.TreeCaches([qkv[..., 128:256]], [qkv[..., 256:]], [k], [v], heads=2)


def chain(B, N):
    return (torch.arange(N, dtype=torch.int32, device="cuda") - 1).repeat(B, 1)


@pytest.mark.parametrize("t", [0.0, 1.0])
def test_accept_ends_where_the_verdict_does(iw, gpu, t):
    """Refused drafts that are drawn again (of draft rows without a distribution), drafts and choices of -1: the caches
    take the accepted drafts and no more, and the next token is the verdict's."""
    print("case: accept follows the verdict", t, flush=True)
    B, N, V = 8, 4, 40
    x = torch.full((B, N, V), -30.0)
    x[:, :, 5] = 9.0  # drawn by any number in the middle
    d = x[:, :N - 1].clone()
    tokens = torch.full((B, N), 5, dtype=torch.int64)
    tokens[:, 0] = 1
    d[0, 0, 3] = math.nan
    d[1, 1] = -math.inf
    d[2, 2, 7] = math.inf
    x[3, 0], tokens[3, 1:] = -math.inf, -1
    x[4, 2, 0], tokens[4, 3] = math.nan, -1
    d[5, 0] = -math.inf
    tokens[6, 2] = -1
    counts = torch.tensor([4, 4, 4, 4, 4, 2, 4, 0], dtype=torch.int32, device="cuda")
    u = torch.full((B, N), 0.5, device="cuda")
    tokens = tokens.cuda()
    got = iw.drafts.verify_drafts(x.cuda(), tokens, d.cuda(), u, counts, temperature=t)
    assert host(got.accepted).tolist() == [0, 1, 2, 0, 2, 0, 1, 0]
    assert host(got.next_token).tolist() == [5, 5, 5, -1, -1, 5, 5, -1]
    lengths = torch.arange(B, dtype=torch.int32, device="cuda")
    acc = caches_of(iw, B, N).accept(tokens, chain(B, N), got.choice, lengths, got.nodes(counts))
    assert host(acc.accepted).tolist() == [1, 2, 3, 1, 3, 1, 2, 0]
    assert torch.equal(acc.next_token[:7], got.next_token[:7])
    assert torch.equal(got.nodes(), got.accepted + 1)


def test_step_without_any_token(iw, gpu):
    """Where every token is suppressed, a step takes the last one alone and has no next token."""
    print("case: step without tokens", flush=True)
    dims, model = small_model(iw)
    B = len(PROMPT)
    mel = iw.synth.synthetic_mel(B, dims.n_mels, 2 * dims.n_audio_ctx, seed=21)
    with torch.no_grad():
        runner = iw.DecoderRunner(model.decoder, B, dims.n_audio_ctx)
        runner.set_audio(model.embed_audio(T(mel)))
        dec = iw.drafts.DraftDecoder(runner, 4, suppress=T(bit_words(range(512), 512)))
        last = dec.start(T(PROMPT), torch.full((B,), 0.5, device="cuda"))
        assert (last == -1).all()
        for i in range(2):
            res = dec.step(last, torch.full((B, 7), 0.5, device="cuda"))
            assert (res.verdict.accepted == 0).all() and (res.verdict.choice == -1).all()
            assert (res.accept.accepted == 1).all() and (res.accept.next_token == -1).all()
            assert (dec.lengths == PROMPT.shape[1] + 1 + i).all()
