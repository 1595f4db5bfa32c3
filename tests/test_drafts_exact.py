"""Sampled decoding at its limits: verdicts that the caches' acceptance follows, log-probabilities of
certain tokens, equal logits at numbers that are their borders, borders as close as a weight is exact, the largest batches."""
import decimal
import math

import numpy as np
import pytest
import torch

from tests import gen
from tests.test_drafts import DTYPES, PROMPT, T, bit_words, drawn_by, host, small_model

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


# Logits (a, m, x, r) and numbers: of rows with a in column 0, m in column 1024, x in the 1023 after that, no r
NEAR = """
0x1.b8f478p-4 -0x1.eb4d6ep+0 -0x1.a4759ap+2 -inf 0x1.a72acap-2
0x1.bb9382p-4 -0x1.eb4d6ep+0 -0x1.a4759ap+2 -inf 0x1.a75378p-2
0x1.06070ep+1 -0x1.4809dp-2 -0x1.57d8dp+2 -inf 0x1.2bf87p-1
-0x1.ac36cp+0 -0x1.c142cap+1 -0x1.08ee9ap+3 -inf 0x1.92d3eep-2
-0x1.6d8c96p-5 -0x1.1c7f48p+1 -0x1.bfdce8p+2 -inf 0x1.e9c4cep-2
-0x1.264ffap+1 -0x1.1f82f2p+2 -0x1.2c321ep+3 -inf 0x1.03bee2p-1
-0x1.367bf8p-2 -0x1.2b7c3ep+1 -0x1.c5c85cp+2 -inf 0x1.c03746p-2
0x1.5c416p+2 0x1.065edp+2 -0x1.503bep+0 -inf 0x1.a16646p-2
0x1.c3f1e8p+2 0x1.33af4p+2 0x1.bb4ap-6 -inf 0x1.fe705ep-2
-0x1.21a412p-1 -0x1.4be7eep+1 -0x1.e54818p+2 -inf 0x1.f3c27cp-2
0x1.71d4d2p+1 0x1.637c64p-3 -0x1.060294p+2 -inf 0x1.fc3d0ap-2
0x1.48b566p+0 -0x1.887744p-1 -0x1.7e3a0ap+2 -inf 0x1.14aaaep-1
0x1.d45662p+2 0x1.60d566p+2 0x1.80dfep-2 -inf 0x1.db94a6p-2
-0x1.520436p-3 -0x1.38375p+1 -0x1.d7deep+2 -inf 0x1.132dcp-1
0x1.cc6642p-1 -0x1.045f58p+0 -0x1.73f99ep+2 -inf 0x1.ac0f4ap-2
-0x1.ef2044p+0 -0x1.c19496p+1 -0x1.14a516p+3 -inf 0x1.a1ab6ap-2
-0x1.419a6cp+0 -0x1.a5c9f4p+1 -0x1.17ed1p+3 -inf 0x1.2d070cp-1
-0x1.7aa9eap+0 -0x1.fdfb6cp+1 -0x1.0fb0ep+3 -inf 0x1.fef0cp-2
0x1.48756ep+1 0x1.a8f366p-4 -0x1.2c2c18p+2 -inf 0x1.1b4fbp-1
0x1.2be034p+0 -0x1.2b7e72p-1 -0x1.84e1b2p+2 -inf 0x1.0d593cp-1
-0x1.51d1ccp+1 -0x1.58679ep+2 -0x1.3cca9cp+3 -inf 0x1.1f19fap-1
-0x1.a0f4ccp+0 -0x1.1e4512p+2 -0x1.12db8ap+3 -inf 0x1.f8cacep-2
"""


# and of rows with a in the first 1024 columns and r in column 2048
FARTHER = """
0x1.63e88cp+2 0x1.b6776cp+2 0x1.5813a4p+2 0x1.d73444p+2 0x1.164802p-1
0x1.22817ep+0 0x1.0458dp+1 0x1.2a1052p+0 0x1.cae124p+1 0x1.f54d96p-2
0x1.033658p+2 0x1.53347ap+2 0x1.dcae92p+1 0x1.08efeep+3 0x1.1dcc6ap-1
0x1.703cccp+1 0x1.1baacp+2 0x1.805c48p+1 0x1.dd36a2p+2 0x1.ca9632p-2
0x1.502036p+0 0x1.1b4198p+2 0x1.1d47ccp+0 0x1.595226p+2 0x1.0d9fe8p-1
0x1.54d118p+1 0x1.d557ap+1 0x1.73d36p+1 0x1.922bbp+2 0x1.bae584p-2
-0x1.c6c0cap-1 0x1.5ac112p+0 -0x1.f680ccp-1 0x1.8232bcp+1 0x1.04318p-1
0x1.2e0104p+2 0x1.67102p+2 0x1.25e01cp+2 0x1.cbc346p+2 0x1.0e5d78p-1
0x1.f2fedep+0 0x1.d29ec8p+1 0x1.f8c4f8p+0 0x1.652edep+2 0x1.f01dcap-2
0x1.70ef16p+2 0x1.e123dcp+2 0x1.77ca94p+2 0x1.1e959p+3 0x1.de3162p-2
0x1.10700cp-1 0x1.9a8d7p+1 0x1.67959p-2 0x1.e0553ap+1 0x1.117618p-1
0x1.c4992ap+0 0x1.4d1b8ep+1 0x1.873a8ep+0 0x1.ab976ep+1 0x1.1d8cc6p-1
-0x1.93098p+0 0x1.a7f2ep-1 -0x1.7033ccp+0 0x1.ac4514p+1 0x1.bf4e6cp-2
0x1.dea006p+1 0x1.310eccp+2 0x1.f1b3c8p+1 0x1.d11262p+2 0x1.d2659ap-2
"""


@pytest.mark.parametrize("copies,rows", [(1, NEAR), (1024, FARTHER)], ids=["two spans", "three spans"])
def test_borders_as_near_as_a_weight_is_exact(iw, gpu, copies, rows):
    """A weight is off by at most 8.2e-13 of itself (the polynomial's 8.14e-13 and the roundings of an exponent and a product), so
    a share s of the whole by less than s (1 - s) 2 * 8.2e-13, at most 4.1e-13, and by the sums' roundings, some 2e-15: numbers
    at 4.3e-13 to 6.1e-13 from a border draw the right one of its tokens."""
    print("case: near borders", copies, flush=True)
    rows = [[float.fromhex(v) for v in line.split()] for line in rows.split("\n") if line]
    x = torch.full((len(rows), 2050), -math.inf)
    want = []
    with decimal.localcontext() as ctx:
        ctx.prec = 40
        for i, (a, m, low, r, u) in enumerate(rows):
            x[i, :copies], x[i, 1024], x[i, 1025:2048], x[i, 2048] = a, m, low, r
            ea, em, el, er = (decimal.Decimal(v).exp() if v > -math.inf else decimal.Decimal(0) for v in (a, m, low, r))
            off = copies * ea / (copies * ea + em + 1023 * el + er) - decimal.Decimal(u)
            assert decimal.Decimal("4.2e-13") < abs(off) < decimal.Decimal("6.5e-13")
            want.append(off > 0)
    got = iw.drafts.sample_tokens(x.cuda(), torch.tensor([r[4] for r in rows], device="cuda"))
    assert [int(v) < 1024 for v in got.tokens] == want


# ---------------------------------------------------------------------------
# sizes
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("N,V,some", [(32, 5, 1 << 20), (64, 3, 1 << 20), (2, 70001, 300)])
def test_verify_as_many_rows_as_a_call_takes(iw, gpu, N, V, some):
    """2^20 rows of one text's logits, of many nodes and of a wide vocabulary."""
    print("case: most rows of drafts", N, V, flush=True)
    B = 1 << 20
    r = gen.rng(N)
    x = torch.from_numpy(r.integers(-12, 13, V).astype(np.int8))
    g = torch.Generator(device="cuda").manual_seed(N)
    u = torch.rand((B, N), generator=g, device="cuda")
    tokens = torch.randint(0, V, (B, N), generator=g, device="cuda")
    if V > 100:
        tokens[:, 1] = int(x.argmax())
    got = iw.drafts.verify_drafts(x.cuda().expand(B, N, V), tokens, None, u, scale=0.25)
    w = np.exp(x.double().numpy() * 0.25)
    p = torch.from_numpy(w / w.sum()).cuda()
    ok = u[:, :-1].double() < p[tokens[:, 1:]]
    taken = ok.long().cumprod(1).sum(1)
    assert torch.equal(got.accepted.long(), taken)
    i = torch.arange(N, device="cuda")
    kept = torch.where(i[:-1] < taken[:, None], tokens[:, 1:], -1)
    assert torch.equal(torch.where(i[:-1] == taken[:, None], -1, got.choice[:, :-1]), kept)
    assert torch.equal(got.choice.gather(1, taken[:, None])[:, 0], got.next_token)
    if some < B:
        for b in np.linspace(0, B - 1, some).astype(int).tolist():
            left = w.copy()
            if int(taken[b]) < N - 1:
                left[int(tokens[b, int(taken[b]) + 1])] = 0
            drawn_by(int(got.next_token[b]), left, float(u[b, N - 1]), left.sum())
        return
    left = p.expand(B, V).clone()
    more = torch.nonzero(taken < N - 1)[:, 0]
    left[more, tokens[more, taken[more] + 1]] = 0
    c = left.cumsum(1)
    at = u[:, -1:].double() * c[:, -1:]
    want = (c <= at).sum(1)
    clear = ((c - at).abs() > 1e-12).all(1)  # numbers that no rounding moves
    assert clear.float().mean() > 0.999 and torch.equal(got.next_token[clear], want[clear])
