"""Sampled decoding at its limits: verdicts that the caches' acceptance follows, log-probabilities of
certain tokens, equal logits at numbers that are their borders."""
import math

import numpy as np
import pytest
import torch

from tests import gen
from tests.test_drafts import DTYPES, PROMPT, T, bit_words, host, small_model

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


# ---------------------------------------------------------------------------
# log-probabilities
# ---------------------------------------------------------------------------

# A lane's suppressed int8 logits are summed with its others and taken off again. A weight has 44 bits, so 64 equal ones have an
# exact sum, and one of 1 among them too where they are 2^-7 or more; less of them leave the sum below 2: 65
# roundings by 2^-53
SUPPRESSED = 66 * 2.0 ** -53


@pytest.mark.parametrize("V", [5, 33, 200, 4096, 4100, 9000])
def test_suppressed_int8_logits_leave_nothing(iw, gpu, V):
    """A row's only token that is not suppressed, at every value and many temperatures, has next to all of the weight."""
    print("case: suppressed int8 logits", V, flush=True)
    at = V // 3
    off = T(bit_words([j for j in range(V) if j != at], V))
    x = torch.full((256, V), -128, dtype=torch.int8, device="cuda")
    x[:, at] = torch.arange(-128, 128).to(torch.int8)
    u = torch.full((256,), 0.5, device="cuda")
    for t in np.linspace(0.05, 40, 60).tolist():
        got = iw.drafts.sample_tokens(x, u, temperature=t, scale=0.5, suppress=off)
        assert (got.tokens == at).all() and float(got.logprob.abs().max()) <= SUPPRESSED, t


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_logprob_is_never_above_0(iw, gpu, dtype):
    """A row's only token has log-probability 0, one that has nearly all of the weight no more than that."""
    print("case: certain tokens", dtype, flush=True)
    values = [0.0, 1.0, -3.25, 5.0, 7.5, -0.4375, 17.0, -30.0, 3.0, 11.0]
    if dtype == "int8":
        values = [0, 1, -3, 5, 127, -128, 17, -30, 64, 99]
    n, low = len(values), -128 if dtype == "int8" else -math.inf
    u = T(gen.rng(2).random(n, np.float32))
    for V in (1, 3, 40, 5000):
        only = torch.full((n, V), low, dtype=DTYPES[dtype])
        at = [(7 * i) % V for i in range(n)]
        for i, v in enumerate(values):
            only[i, at[i]] = v
        for t in (1.0, 0.7, 0.01, 0.0):
            # the token alone; int8 rows, whose lowest value is a logit like others, with all others suppressed
            for i in range(n):
                off = None if dtype != "int8" or V == 1 else T(bit_words([j for j in range(V) if j != at[i]], V))
                got = iw.drafts.sample_tokens(only[i:i + 1].cuda(), u[i:i + 1], temperature=t, scale=0.5, suppress=off)
                lp = float(got.logprob[0])
                assert int(got.tokens[0]) == at[i]
                assert lp == 0.0 if off is None else -SUPPRESSED <= lp <= 0.0, (V, t, values[i], lp)
    if dtype == "int8":
        x = torch.full((256, 200), -128, dtype=torch.int8, device="cuda")
        x[:, 66] = torch.arange(-128, 128).to(torch.int8)
        off = T(bit_words([j for j in range(200) if j != 66], 200))
        for t in np.linspace(0.05, 40, 60).tolist():
            got = iw.drafts.sample_tokens(x, torch.full((256,), 0.5, device="cuda"), temperature=t, scale=0.5, suppress=off)
            assert (got.logprob <= 0).all(), t
    V = 3001
    x = torch.from_numpy(gen.rng(3).normal(0, 1, (64, V)))
    x[:, 11] = torch.linspace(10, 60, 64)
    scale = 0.5 if dtype == "int8" else 1.0
    x = (x / scale).round().clamp(-127, 127).to(torch.int8) if dtype == "int8" else x.to(DTYPES[dtype])
    got = iw.drafts.sample_tokens(x.cuda(), torch.full((64,), 0.3, device="cuda"), scale=scale)
    assert (got.tokens == 11).all() and (got.logprob <= 0).all()


# ---------------------------------------------------------------------------
# borders
# ---------------------------------------------------------------------------

def drawn_either_way(iw, x, u, t):
    """Tokens of rows by sample_tokens, and as the tokens after chains of no drafts."""
    last = torch.zeros((len(u), 1), dtype=torch.int64, device="cuda")
    return (iw.drafts.sample_tokens(x, u, temperature=t).tokens,
            iw.drafts.verify_drafts(x[:, None], last, None, u[:, None], temperature=t).next_token)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("apart", [1, 37, 1100, 5000])
def test_equal_logits_share_exactly(iw, gpu, apart, dtype):
    """Two to sixteen equal logits in a row of less likely ones: a number that is the border of two of them draws the
    second, the one before it the first."""
    print("case: equal logits", apart, dtype, flush=True)
    values = [0, -3, 1, 64, 127, -100] if dtype == "int8" else [0.0, -3.25, 1.0, 5.0, 7.5, 0.28125, -11.0]
    for k in (2, 4, 8, 16):
        V = apart * k + 3
        x = torch.full((len(values), V), -127 if dtype == "int8" else -math.inf, dtype=DTYPES[dtype])
        for i, v in enumerate(values):
            x[i, 2:2 + apart * k:apart] = v
        j = torch.arange(k, dtype=torch.float32)
        u = torch.stack([j / k, torch.nextafter((j + 1) / k, torch.zeros(k))], 1).reshape(-1)
        want = (2 + apart * j.long()).repeat_interleave(2)
        for t in ((0.001,) if dtype == "int8" else (1.0, 0.7, 3.0)):  # int8: the others' weights are 0
            for row in x:
                for got in drawn_either_way(iw, row.cuda().expand(2 * k, V), u.cuda(), t):
                    assert torch.equal(got.cpu(), want), (k, t, float(row.max()), got.tolist())


@pytest.mark.parametrize("k", [3, 5, 6, 7, 10, 12, 24, 100])
def test_equal_int8_logits_of_any_number_share_exactly(iw, gpu, k):
    print("case: equal int8 logits", k, flush=True)
    x = torch.full((1, 900), -127, dtype=torch.int8)
    x[0, 5:5 + 7 * k:7] = 3
    j = torch.arange(64)
    for got in drawn_either_way(iw, x.cuda().expand(64, 900), (j / 64).cuda(), 0.001):
        assert torch.equal(got.cpu(), 5 + 7 * (j * k // 64))
