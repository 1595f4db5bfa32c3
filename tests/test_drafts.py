"""Sampled decoding with drafts on the GPU against plain implementations.

* window_attention: bit-exact with the CPU oracle's attention under a mask of the
  visible keys (tile borders, V layouts, projected rows, ragged lengths and counts, given
  positions, empty rows, wrapping row maxima, every frac_bits)
* sample_tokens, verify_drafts: distribution functions in float64 on the host
* DraftDecoder: greedy decoding's tokens at temperature 0, every draft accepted where
  it saw all keys, the caches of a decoder that was given the tokens
"""
import math

import numpy as np
import pytest
import torch

from tests import gen

pytestmark = pytest.mark.gpu


def T(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def host(t):
    return t.cpu().numpy()


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

class Window:
    """Random operands; keys and values past the rows' lengths are noise."""

    def __init__(self, seed, B, H, D, cap, N, before, after=0, sinks=0, lengths=None, counts=None, positions=None,
                 layout="vt", scalars=None, k_rows=False):
        r = gen.rng(seed)
        self.B, self.H, self.D, self.cap, self.N, self.layout = B, H, D, cap, N, layout
        self.before, self.after, self.sinks = before, after, sinks
        C = H * D
        _, _, _, qm, qs, f, am, as_ = gen.attn_case(seed, 1, 1, 1, 1, D)
        self.sc = scalars or (qm, qs, f, am, as_)
        self.q = gen.i8(r, (B, N, 3 * C), -127, 127)
        self.k = gen.i8(r, (B, H, cap, D), -127, 127)
        self.v = gen.i8(r, (B, H, D, cap), -127, 127)
        self.lengths = None if lengths is None else np.asarray(lengths, np.int32)
        self.counts = None if counts is None else np.asarray(counts, np.int32)
        self.positions = None if positions is None else np.asarray(positions, np.int32)
        shape, self.vs = gen.v_cache_layout(B, H, D, cap, layout)
        self.vc = gen.i8(r, shape)
        gen.v_cache_put(self.vc, layout, 0, self.v)
        self.k_rows = k_rows

    def v_view(self, vc):
        D = self.D
        if self.layout == "vt":
            return vc
        nq = vc.shape[2]
        return vc[..., :4 * D].unflatten(3, (D, 4)) if vc.shape[3] > 4 * D else vc.view(self.B, self.H, nq, D, 4)

    def args(self):
        C = self.H * self.D
        k = T(self.k)
        if self.k_rows:  # the middle columns of a projection's rows
            rows = torch.zeros((self.B, self.cap, 3 * C), dtype=torch.int8, device="cuda")
            rows[..., C:2 * C] = k.transpose(1, 2).flatten(2)
            k = rows[..., C:2 * C].unflatten(2, (self.H, self.D)).transpose(1, 2)
        opt = lambda a: None if a is None else T(a)
        return [T(self.q)[..., :C], k, self.v_view(T(self.vc)), opt(self.lengths)], dict(
            positions=opt(self.positions), counts=opt(self.counts))

    def kw(self):
        qm, qs, f, am, as_ = self.sc
        return dict(heads=self.H, before=self.before, after=self.after, sinks=self.sinks, qk_multiplier=qm, qk_shift=qs,
                    frac_bits=f, av_multiplier=am, av_shift=as_)

    def run(self, iw, **kw):
        args, opt = self.args()
        return iw.drafts.window_attention(*args, **opt, **self.kw(), **kw)

    def hidden(self, b):
        """(length, count, [count, length] hidden keys) of a row."""
        ln = self.cap if self.lengths is None else min(max(int(self.lengths[b]), 0), self.cap)
        cnt = self.N if self.counts is None else min(max(int(self.counts[b]), 0), self.N)
        p = (ln - cnt + np.arange(cnt) if self.positions is None else self.positions[b, :cnt].astype(np.int64))[:, None]
        far = 1 << 40
        before, after = (far if x is None else x for x in (self.before, self.after))
        j = np.arange(ln)
        return ln, cnt, ~((j <= p + after) & ((j >= p - before) | (j < self.sinks)))

    def expected(self, oracle, rows=None):
        B, H, D, N, C = self.B, self.H, self.D, self.N, self.H * self.D
        out = np.zeros((B, N, C), np.int8)
        for b in range(B) if rows is None else rows:
            ln, cnt, hidden = self.hidden(b)
            if cnt == 0 or ln == 0:
                continue
            q = self.q[b, :cnt, :C].reshape(cnt, H, D).transpose(1, 0, 2)
            y = oracle.attention(np.ascontiguousarray(q[None]), np.ascontiguousarray(self.k[b:b + 1, :, :ln]),
                                 np.ascontiguousarray(self.v[b:b + 1, :, :, :ln]), np.ascontiguousarray(hidden), *self.sc)[0]
            y[hidden.all(1)] = 0
            out[b, :cnt] = y
        return out

    def check(self, iw, oracle, **kw):
        got, want = host(self.run(iw, **kw)), self.expected(oracle)
        bad = np.argwhere(got != want)
        assert not len(bad), (len(bad), bad[:4])


LAYOUTS = ("vt", "quads", "quads_pad")


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("N", [1, 2, 5, 15, 16, 17, 31, 32, 33, 64, 65, 130])
def test_window_queries(iw, oracle, gpu, N, layout):
    print("case: window queries", N, layout, flush=True)
    Window(7 * N, 3, 2, 64, 200, N, 40, 0, 3, lengths=[200, N, 131], layout=layout).check(iw, oracle)


@pytest.mark.parametrize("layout", ["vt", "quads"])
@pytest.mark.parametrize("D", [16, 32, 48, 64, 80, 96, 112, 128])
def test_window_head_dims(iw, oracle, gpu, D, layout):
    print("case: window head dim", D, layout, flush=True)
    Window(D, 2, 3, D, 300, 21, 70, 5, 2, lengths=[300, 77], counts=[21, 20], layout=layout).check(iw, oracle)


@pytest.mark.parametrize("layout", ["vt", "quads"])
@pytest.mark.parametrize("length", [0, 1, 2, 3, 4, 5, 15, 16, 17, 63, 64, 65, 127, 128, 129, 191, 192, 193, 447, 448])
def test_window_lengths(iw, oracle, gpu, length, layout):
    """Key counts that end inside a quad, a product, a chunk or the cache, for one token and a few."""
    print("case: window length", length, layout, flush=True)
    for N in (1, 6):
        Window(3 * length + N, 2, 4, 64, 448, N, 100, 0, 4, lengths=[length, 448 - length], layout=layout).check(iw, oracle)


@pytest.mark.parametrize("before,after,sinks", [
    (0, 0, 0), (0, 0, 1), (0, 0, 500), (1, 0, 0), (15, 0, 16), (16, 16, 0), (63, 0, 64), (64, 0, 65), (65, 64, 63), (5, 300, 0),
    (300, 0, 0), (None, 0, 0), (None, None, 0), (0, None, 0), (10, None, 3), (2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1)])
def test_window_widths(iw, oracle, gpu, before, after, sinks):
    print("case: window width", before, after, sinks, flush=True)
    for N in (1, 50, 260):
        Window(11, 2, 2, 64, 260, N, before, after, sinks, lengths=[260, 201], layout="quads").check(iw, oracle)


@pytest.mark.parametrize("layout", ["vt", "quads"])
def test_window_positions(iw, oracle, gpu, layout):
    """Given positions: in any order, before the first key, behind the last, at the ends of 32 bits."""
    print("case: window positions", layout, flush=True)
    r = gen.rng(5)
    B, N, cap = 4, 37, 500
    p = r.integers(-50, cap + 50, (B, N))
    p[1] = np.sort(p[1])
    p[2, :8] = [-2 ** 31, 2 ** 31 - 1, -1, 0, cap - 1, cap, cap + 39, cap + 41]
    for before, after, sinks in ((40, 0, 0), (40, 60, 5), (0, 0, 70), (None, 3, 0), (2 ** 31 - 1, 2 ** 31 - 1, 0)):
        Window(6, B, 2, 64, cap, N, before, after, sinks, lengths=[cap, 480, cap, 3], counts=[N, N - 1, N, 20], positions=p,
               layout=layout).check(iw, oracle)
        Window(7, B, 2, 64, cap, 1, before, after, sinks, lengths=[cap, 480, cap, 3], positions=p[:, 2:3],
               layout=layout).check(iw, oracle)


@pytest.mark.parametrize("N,before,after,sinks", [(500, 31, 31, 0), (500, 127, 127, 16), (333, 100, 0, 70), (1500, 255, 255, 4)])
def test_window_local_rows(iw, oracle, gpu, N, before, after, sinks):
    """Every position of a sequence, the keys as columns of the projection's rows."""
    print("case: window rows", N, before, after, flush=True)
    Window(N, 1, 3, 64, N, N, before, after, sinks, k_rows=True).check(iw, oracle)


@pytest.mark.parametrize("layout", ["vt", "quads"])
@pytest.mark.parametrize("D,B,N,before,after,sinks", [
    (64, 260, 33, 100, 0, 3), (48, 260, 64, 17, 40, 70), (64, 129, 70, 63, 64, 0), (16, 256, 48, 250, 250, 1),
    (128, 130, 40, 63, 0, 4), (80, 128, 64, 30, 31, 0), (112, 65, 65, 200, 3, 80),
    (64, 130, 33, 448, 0, 20), (32, 65, 129, 300, 200, 0), (128, 130, 50, 449, 0, 0), (96, 64, 200, 200, 260, 100),
    (128, 64, 257, None, 0, 0)])
def test_window_many_rows(iw, oracle, gpu, D, B, N, before, after, sinks, layout):
    """Batches whose queries share keys: ragged lengths and counts, rows without either, every path of the scalars."""
    print("case: window many rows", D, B, N, before, after, sinks, layout, flush=True)
    r = gen.rng(B + N + D)
    cap = 600
    lengths = r.integers(0, cap + 1, B)
    counts = r.integers(0, N + 1, B)
    lengths[:6], counts[:6] = [cap, cap - 1, 0, 1, 300, N], [N, N - 1, N, N, 0, N]
    rows = [0, 1, 2, 3, 4, 5, B // 2, B - 2, B - 1]
    for scalars in (None, (255, 0, 7, 130, 9), (200, 4, 10, 255, 12), (3, 9, 12, 90, 7)):
        w = Window(D + N, B, 2, D, cap, N, before, after, sinks, lengths=lengths, counts=counts, layout=layout, scalars=scalars)
        got, want = host(w.run(iw)), w.expected(oracle, rows)
        bad = np.argwhere(got[rows] != want[rows])
        assert not len(bad), (scalars, len(bad), bad[:4])
        unused = np.arange(N) >= np.asarray(counts)[:, None]
        assert not got[unused].any()


@pytest.mark.parametrize("B,H,D,cap,N", [(1, 20, 64, 300, 300), (40, 20, 64, 100, 7), (129, 3, 64, 100, 40), (16, 20, 64, 130, 100),
                                         (24, 20, 96, 130, 100), (9, 16, 128, 260, 200), (2, 2, 64, 2000, 1500), (130, 20, 64, 448, 1),
                                         (700, 8, 64, 150, 33)])
def test_window_grids(iw, oracle, gpu, B, H, D, cap, N):
    """Few and many blocks: the forms that the sizes choose."""
    print("case: window grid", B, H, D, cap, N, flush=True)
    r = gen.rng(B)
    c = Window(B + N, B, H, D, cap, N, 90, 10, 2, lengths=r.integers(0, cap + 1, B), counts=r.integers(0, N + 1, B),
               layout="quads" if B % 2 else "vt")
    some = sorted({0, 1, B // 2, B - 2, B - 1} & set(range(B)))
    got, want = host(c.run(iw)), c.expected(oracle, some)
    for b in some:
        assert np.array_equal(got[b], want[b]), b


@pytest.mark.parametrize("layout", ["vt", "quads"])
@pytest.mark.parametrize("D,cap,N,before", [(64, 9000, 1, 4095), (128, 9000, 1, 4095), (128, 5000, 8, 2047), (96, 4500, 17, 4400),
                                            (64, 20000, 3, 16000), (112, 6000, 33, 3000)])
def test_window_long(iw, oracle, gpu, D, cap, N, before, layout):
    """Few heads over wide windows of long caches."""
    print("case: window long", D, cap, N, layout, flush=True)
    for lengths in ([cap, 700], [cap - 77, 0], [1, cap // 2]):
        Window(N + D, 2, 2, D, cap, N, before, 0, 70, lengths=lengths, counts=[N, max(1, N - 1)], layout=layout).check(iw, oracle)


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("D", [16, 48, 64, 80, 128])
@pytest.mark.parametrize("cap,before,after,sinks", [
    (64, 15, 0, 0), (200, 0, 0, 1), (333, 127, 0, 4), (900, 100, 100, 20), (900, 400, 3, 0), (1500, 1000, 200, 40),
    (1000, None, None, 0), (6000, 4500, 0, 33)])
def test_window_one_query(iw, oracle, gpu, cap, before, after, sinks, D, layout):
    """A token a row: first keys inside the window and beside it, positions before the first key and behind the last."""
    print("case: window one query", cap, before, after, sinks, D, layout, flush=True)
    r = gen.rng(cap + D)
    lengths = [cap, cap - 1, 0, 1, 17, cap // 2, cap // 2 + 1, cap]
    counts = [1, 1, 1, 1, 1, 1, 1, 0]
    positions = [[cap - 1], [-5], [3], [0], [40], [cap // 3], [2 ** 31 - 1], [5]]
    for given in (None, positions):
        for scalars in (None, (255, 0, 7, 130, 9), (1, 0, 13, 90, 3)):
            Window(int(r.integers(1 << 20)), 8, 2, D, cap, 1, before, after, sinks, lengths=lengths, counts=counts,
                   positions=given, layout=layout, scalars=scalars).check(iw, oracle)


@pytest.mark.parametrize("layout", ["vt", "quads"])
@pytest.mark.parametrize("D,B,cap", [(16, 66, 16000), (80, 33, 16000), (64, 260, 700)])
def test_window_one_query_many_heads(iw, oracle, gpu, D, B, cap, layout):
    """A token of many rows, over more keys than a block keeps scores of too."""
    print("case: window one query many heads", D, B, cap, layout, flush=True)
    r = gen.rng(cap + D)
    lengths = r.integers(0, cap + 1, B)
    lengths[0] = cap
    w = Window(D + B, B, 4, D, cap, 1, cap - 1000 if cap > 1000 else None, 0, 10, lengths=lengths, layout=layout)
    rows = [0, 1, B // 2, B - 1]
    got, want = host(w.run(iw)), w.expected(oracle, rows)
    assert (got[rows] == want[rows]).all()


@pytest.mark.parametrize("f", range(1, 14))
@pytest.mark.parametrize("qk", [(255, 0), (1, 0), (200, 4), (3, 9), (255, 31), (255, 40), (0, 3)])
def test_window_scalars(iw, oracle, gpu, f, qk):
    """Row maxima that saturate and wrap, every precision of the shift exponential."""
    print("case: window scalars", f, qk, flush=True)
    for N in (1, 40):
        Window(f, 1, 2, 64, 150, N, 60, 3, 2, lengths=[150], scalars=(*qk, f, 200, 7)).check(iw, oracle)


@pytest.mark.parametrize("av", [(255, 0), (1, 0), (130, 9), (255, 32), (255, -3)])
def test_window_output_scalars(iw, oracle, gpu, av):
    print("case: window output scalars", av, flush=True)
    Window(3, 1, 2, 80, 150, 9, 60, 3, 2, scalars=(120, 8, 8, *av)).check(iw, oracle)


def test_window_clamps_lengths_and_counts(iw, oracle, gpu):
    print("case: window clamps", flush=True)
    Window(4, 3, 2, 64, 90, 9, 30, 0, 1, lengths=[-5, 2 ** 30, 91], counts=[9, 2 ** 30, -1]).check(iw, oracle)


def test_window_out(iw, oracle, gpu):
    """The result in the place of q, and between columns of the rows that the keys lie in."""
    print("case: window out", flush=True)
    c = Window(9, 2, 3, 64, 120, 120, 40, 40, 2, k_rows=True)
    want = c.expected(oracle)
    C = c.H * c.D
    for where in (0, 2):
        rows = torch.zeros((2, 120, 3 * C), dtype=torch.int8, device="cuda")
        rows[..., :C] = T(c.q)[..., :C]
        rows[..., C:2 * C] = T(c.k).transpose(1, 2).flatten(2)
        k = rows[..., C:2 * C].unflatten(2, (c.H, c.D)).transpose(1, 2)
        out = rows[..., where * C:(where + 1) * C]
        got = iw.drafts.window_attention(rows[..., :C], k, T(c.vc), out=out, **c.kw())
        assert got is out and np.array_equal(host(got), want)
        assert torch.equal(k, T(c.k))


def test_window_equals_tree_attention(iw, gpu):
    """One token over a cache that holds it already, without a window: the tree's one node."""
    print("case: window and tree", flush=True)
    r = gen.rng(3)
    B, H, D, cap = 3, 4, 64, 200
    C = H * D
    qkv = T(gen.i8(r, (B, 1, 3 * C)))
    k, v = T(gen.i8(r, (B, H, cap, D))), T(gen.i8(r, (B, H, cap // 4, D, 4)))
    ln = T(np.array([0, 77, 199], np.int32))
    sc = dict(heads=H, qk_multiplier=90, qk_shift=9, frac_bits=8, av_multiplier=100, av_shift=6)
    want = iw.speculative.tree_attention(qkv[..., :C], qkv[..., C:2 * C], qkv[..., 2 * C:], k, v, ln,
                                         torch.ones((B, 1), dtype=torch.int64, device="cuda"), **sc)
    tok = torch.zeros((B, 1), dtype=torch.int64, device="cuda")
    iw.speculative.TreeCaches([qkv[..., C:2 * C]], [qkv[..., 2 * C:]], [k], [v], heads=H).accept(
        tok, tok.int() - 1, tok, ln)
    got = iw.drafts.window_attention(qkv[..., :C], k, v, ln + 1, before=None, **sc)
    assert torch.equal(got, want)


def test_window_equals_the_masked_attention(iw, oracle, gpu):
    """An encoder's local attention and the prefill kernel under the same mask."""
    print("case: window and prefill", flush=True)
    c = Window(13, 2, 4, 64, 700, 700, 100, 100, 8)
    hidden = c.hidden(0)[2]
    got = host(c.run(iw))
    C = c.H * c.D
    q = c.q[..., :C].reshape(2, 700, c.H, c.D).transpose(0, 2, 1, 3)
    want = oracle.attention(np.ascontiguousarray(q), c.k, c.v, np.ascontiguousarray(hidden), *c.sc)
    assert np.array_equal(got, want)


# ---------------------------------------------------------------------------
# tokens
# ---------------------------------------------------------------------------

DTYPES = {"int8": torch.int8, "float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def make_logits(r, shape, dtype, scale=0.125):
    """Logits as a model leaves them (CPU): a few candidates stand out."""
    V = shape[-1]
    x = r.normal(-4, 2, shape).reshape(-1, V)
    for row in x:
        row[r.integers(0, V, min(5, V))] += r.uniform(3, 16, min(5, V))
    x = torch.from_numpy(x.reshape(shape))
    if dtype == "int8":
        return (x / scale).round().clamp(-127, 127).to(torch.int8)
    return x.to(DTYPES[dtype])


def bit_words(ids, V):
    w = np.zeros((V + 31) // 32, np.uint32)
    for i in ids:
        w[i >> 5] |= np.uint32(1) << np.uint32(i & 31)
    return w.view(np.int32)


def weights(x, scale, t, suppress=()):
    """Weights of one row in float64 on the host, the largest 1; None without a distribution."""
    x = x.double().numpy().copy()
    x[list(suppress)] = -np.inf
    m = x.max()
    if not np.isfinite(m):
        return None
    if not t > 0:
        w = np.zeros_like(x)
        w[x.argmax()] = 1.0
        return w
    return np.exp((x - m) * (scale / t))


def drawn_by(tok, w, u, scale_of=1.0):
    """tok is the token that u draws from w. A weight is off by 7.8e-13 of itself (the polynomial) and its exponent's
    rounding (|t| 2^t 2^-52 < 2^-52 of the largest, t = log2 w), a sum by one rounding a term: a border and the whole that
    it is a share of by less than 2 * 7.8e-13 + (V + 100) 2^-52 of the whole."""
    u = min(max(float(u), 0.0), 1 - 2.0 ** -24)
    c = np.cumsum(w)
    room = (2 * 7.8e-13 + (len(w) + 100) * 2.0 ** -52) * scale_of
    assert 0 <= tok < len(w) and w[tok] > 0, tok
    assert c[tok] - w[tok] <= u * c[-1] + room and c[tok] > u * c[-1] - room, (tok, c[tok], u * c[-1])


def check_samples(got, logits, u, t, scale, suppress=()):
    t = np.broadcast_to(t, len(u))
    for r in range(len(u)):
        w = weights(logits[r], scale, float(t[r]), suppress)
        tok, lp = int(got.tokens[r]), float(got.logprob[r])
        if w is None:
            assert tok == -1 and math.isnan(lp), r
            continue
        drawn_by(tok, w, u[r], w.sum())
        want = math.log(w[tok] / w.sum())
        # rounded once to float32, from numbers of 64 bits
        assert abs(lp - want) <= 2.0 ** -24 * abs(want) + 1e-12, (r, lp, want)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,V", [(1, 1), (2, 2), (3, 3), (5, 31), (5, 33), (4, 255), (4, 256), (3, 257), (2, 1000), (2, 4095),
                                    (2, 4097), (3, 8200), (130, 1025), (2, 51865), (1, 262147), (3, 70001)])
def test_sample_tokens(iw, gpu, rows, V, dtype):
    print("case: sample", rows, V, dtype, flush=True)
    r = gen.rng(rows + V)
    x = make_logits(r, (rows, V), dtype)
    u = r.random(rows, np.float32)
    scale = 0.125 if dtype == "int8" else 1.0
    for t in (1.0, 0.3):
        check_samples(iw.drafts.sample_tokens(x.cuda(), T(u), temperature=t, scale=scale), x, u, t, scale)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_sample_every_border(iw, gpu, dtype):
    """Numbers right at and beside the borders of the distribution function, every token drawn."""
    print("case: sample borders", dtype, flush=True)
    V = 400
    r = gen.rng(2)
    x = make_logits(r, (1, V), dtype)
    scale = 0.02 if dtype == "int8" else 0.3
    w = weights(x[0], scale, 1.0)
    c = np.cumsum(w) / w.sum()
    u = np.concatenate([c - 1e-5, c + 1e-5, [0.0, 1.0, 2.0, -1.0, np.nan, np.inf, -np.inf]]).astype(np.float32)
    got = iw.drafts.sample_tokens(x.cuda().expand(len(u), V), T(u), scale=scale)
    check_samples(got, x.expand(len(u), V), np.nan_to_num(u, nan=0.0, posinf=1.0, neginf=0.0), 1.0, scale)
    assert len(set(host(got.tokens))) > V // 2


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("shift", [0, 1, 3, 7, 15])
def test_sample_strides(iw, gpu, shift, dtype):
    """Rows at every alignment, padded and reordered; leading dims kept."""
    print("case: sample strides", shift, dtype, flush=True)
    r = gen.rng(shift)
    V, rows = 5003, 6
    x = make_logits(r, (rows, V), dtype)
    u = r.random(rows, np.float32)
    scale = 0.125 if dtype == "int8" else 1.0
    want = iw.drafts.sample_tokens(x.cuda(), T(u), scale=scale)
    check_samples(want, x, u, 1.0, scale)
    wide = torch.full((rows, V + 40), 100, dtype=x.dtype, device="cuda")
    wide[:, shift:shift + V] = x.cuda()
    columns = x.t().contiguous().cuda().t()
    for y, v in ((wide[:, shift:shift + V], T(u)), (columns, T(u)), (x.cuda().view(2, 3, V), T(u).view(2, 3))):
        got = iw.drafts.sample_tokens(y, v, scale=scale)
        assert got.tokens.shape == v.shape
        assert torch.equal(got.tokens.flatten(), want.tokens) and torch.equal(got.logprob.flatten(), want.logprob)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("V", [40, 5000, 70001])
def test_sample_suppressed(iw, gpu, V, dtype):
    """Suppressed tokens are never drawn, at any temperature, whatever their logits."""
    print("case: sample suppressed", V, dtype, flush=True)
    r = gen.rng(V)
    x = make_logits(r, (9, V), dtype)
    off = sorted(set(r.integers(0, V, 30).tolist()) | {0, V - 1} | set(x.double().argmax(1).tolist()))
    off = [i for i in off if i != 7]
    u = r.random(9, np.float32)
    u[0] = 0.0
    scale = 0.125 if dtype == "int8" else 1.0
    for t in (1.0, 0.0, 0.01):
        got = iw.drafts.sample_tokens(x.cuda(), T(u), temperature=t, scale=scale, suppress=T(bit_words(off, V)))
        check_samples(got, x, u, t, scale, off)
    none = iw.drafts.sample_tokens(x.cuda(), T(u), scale=scale, suppress=T(bit_words(range(V), V)))
    assert (none.tokens == -1).all() and none.logprob.isnan().all()


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_sample_temperatures_of_rows(iw, gpu, dtype):
    """A temperature of each row, 0 among them (the first of the largest), and odd ones."""
    print("case: sample temperatures", dtype, flush=True)
    r = gen.rng(8)
    t = np.array([0.0, 0.2, 1.0, 5.0, 1e-30, 1e-3, 1e30, np.inf, -1.0, np.nan, 0.0, 0.8], np.float32)
    V = 9001
    x = make_logits(r, (len(t), V), dtype)
    x[0, [5, 77, 4444, 8999]] = x[0].max()
    x[10] = x[10].max()
    scale = 0.125 if dtype == "int8" else 1.0
    u = r.random(len(t), np.float32)
    got = iw.drafts.sample_tokens(x.cuda(), T(u), temperature=T(t), scale=scale)
    ref = np.where(t > 0, t, 0)
    check_samples(got, x, u, np.where(np.isinf(ref), 1e300, ref.astype(np.float64)), scale)
    assert int(got.tokens[0]) == int(x[0].double().argmax()) and int(got.tokens[10]) == 0


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("t,scale", [(5e-324, 1.0), (1e-310, 2.0 ** 100), (1e-300, 1e-30), (2.0 ** 100, 1e-300)])
def test_sample_extreme_temperatures(iw, gpu, t, scale, dtype):
    """Next to no temperature leaves the largest logits, in equal shares; one that is all too high, all logits."""
    print("case: sample extreme temperatures", t, scale, dtype, flush=True)
    V, ties = 1000, [3, 500, 998, 999]
    x = torch.full((64, V), -7.0)
    x[:, ties] = 5.0
    u = ((torch.arange(64) + 0.5) / 64).cuda()
    got = iw.drafts.sample_tokens(x.to(DTYPES[dtype]).cuda(), u, temperature=t, scale=scale)
    low = t > 1
    want = [int((i + 0.5) / 64 * V) if low else ties[i // 16] for i in range(64)]
    assert host(got.tokens).tolist() == want
    assert np.allclose(host(got.logprob), -math.log(V if low else 4), rtol=1e-6, atol=0)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("V", [20, 3000, 70001])
def test_sample_special_values(iw, gpu, V, dtype):
    """-inf is never drawn; rows with NaN, +inf or nothing finite have no token."""
    print("case: sample special", V, dtype, flush=True)
    r = gen.rng(V)
    x = make_logits(r, (10, V), dtype)
    x[0, :V - 1] = -math.inf
    x[1] = -math.inf
    x[2, V // 2] = math.inf
    x[3, V - 1] = math.nan
    x[4, 0] = -math.nan
    x[5, ::2] = -math.inf
    x[6] = torch.finfo(x.dtype).min
    x[7] = torch.finfo(x.dtype).min
    x[7, 3] = torch.finfo(x.dtype).max
    x[8, 1:] = torch.finfo(x.dtype).min
    for uv in (0.0, 0.5, 0.999999):
        u = np.full(10, uv, np.float32)
        for t in (1.0, 0.0):
            got = iw.drafts.sample_tokens(x.cuda(), T(u), temperature=t)
            check_samples(got, x, u, t, 1.0)


def test_sample_distribution(iw, gpu):
    """Of 2^18 draws each token comes up as often as its probability says, within six deviations."""
    print("case: sample distribution", flush=True)
    n, V = 1 << 18, 24
    r = gen.rng(1)
    x = torch.from_numpy(r.normal(0, 1.5, V)).float()
    got = iw.drafts.sample_tokens(x.cuda().expand(n, V), T(r.random(n, np.float32)), temperature=0.7)
    p = torch.softmax(x.double() / 0.7, 0).numpy()
    f = np.bincount(host(got.tokens), minlength=V) / n
    assert (np.abs(f - p) <= 6 * np.sqrt(p * (1 - p) / n)).all()


# ---------------------------------------------------------------------------
# drafts
# ---------------------------------------------------------------------------

def check_verdict(got, logits, tokens, draft, u, counts, t, scale, dt=None, dscale=None, suppress=()):
    B, N, V = logits.shape
    choice, accepted, nxt = (host(x) for x in got)
    t = np.broadcast_to(t, B)
    dt = t if dt is None else np.broadcast_to(dt, B)
    dscale = scale if dscale is None else dscale
    clamp = lambda v: min(max(float(v), 0.0), 1 - 2.0 ** -24) if v == v else 0.0
    for b in range(B):
        cnt = N if counts is None else min(max(int(counts[b]), 0), N)
        a, left, ok = 0, None, cnt > 0
        while ok:
            p = weights(logits[b, a], scale, float(t[b]), suppress)
            if p is None:
                break
            p = p / p.sum()
            left = p
            if a + 1 >= cnt:
                break
            x = int(tokens[b, a + 1])
            inside = 0 <= x < V
            if draft is None:
                q, has = np.zeros(V), True
                if inside:
                    q[x] = 1.0
                qx = 1.0
            else:
                q = weights(draft[b, a], dscale, float(dt[b]), suppress)
                has = q is not None
                if has:
                    q = q / q.sum()
                    qx = q[x] if inside else 0.0
            if has and clamp(u[b, a]) * qx < (p[x] if inside else 0.0):
                a += 1
                left = None
                continue
            if has:
                rest = np.maximum(p - q, 0)
                # probabilities that are equal but for their last bits leave nothing
                rest[np.abs(p - q) < 1e-14 * p] = 0
                left = rest if rest.sum() > 0 else p
            break
        assert accepted[b] == a, (b, accepted[b], a)
        want = np.full(N, -1)
        want[:a] = host(tokens)[b, 1:a + 1]
        if left is None:
            assert nxt[b] == -1, b
        else:
            drawn_by(int(nxt[b]), left, clamp(u[b, N - 1]))
            want[a] = nxt[b]
        assert np.array_equal(choice[b], want), (b, choice[b], want)


def make_drafts(r, B, N, V, dtype, scale, t, noise=1.0, drawn=True):
    """Target logits, weaker draft logits, tokens drawn from those (CPU), numbers."""
    x = make_logits(r, (B, N, V), "float32").double()
    d = x[:, :N - 1] + torch.from_numpy(r.normal(0, noise, (B, N - 1, V)))
    conv = (lambda y: (y / scale).round().clamp(-127, 127).to(torch.int8)) if dtype == "int8" else (lambda y: y.to(DTYPES[dtype]))
    x, d = conv(x), conv(d)
    tt = torch.from_numpy(np.broadcast_to(np.asarray(t, np.float64), B).copy())[:, None, None]
    g = torch.from_numpy(r.gumbel(size=(B, N - 1, V)))
    tokens = torch.zeros((B, N), dtype=torch.int64)
    tokens[:, 1:] = (d.double() * scale + g * tt).argmax(-1)
    return x, d, tokens, r.random((B, N), np.float32)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("B,N,V", [(1, 1, 1), (2, 2, 2), (3, 1, 700), (3, 4, 31), (5, 6, 1000), (2, 3, 4097), (1, 5, 51865), (9, 16, 300),
                                   (2, 64, 513), (70, 3, 1030), (1, 2, 262147)])
def test_verify_drafts(iw, gpu, B, N, V, dtype):
    print("case: verify", B, N, V, dtype, flush=True)
    r = gen.rng(B + N + V)
    scale = 0.125 if dtype == "int8" else 1.0
    x, d, tokens, u = make_drafts(r, B, N, V, dtype, scale, 0.7)
    counts = np.where(r.random(B) < 0.3, r.integers(0, N + 1, B), N).astype(np.int32)
    for draft in (d, None):
        for cnt in (counts, None):
            got = iw.drafts.verify_drafts(x.cuda(), tokens.cuda(), None if draft is None else draft.cuda(), T(u),
                                          None if cnt is None else T(cnt), temperature=0.7, scale=scale)
            check_verdict(got, x, tokens, draft, u, cnt, 0.7, scale)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_verify_temperatures(iw, gpu, dtype):
    """Rows at temperatures of their own, 0 on either side or both, drafts at another temperature and scale."""
    print("case: verify temperatures", dtype, flush=True)
    r = gen.rng(5)
    B, N, V = 24, 5, 3001
    scale = 0.125 if dtype == "int8" else 1.0
    t = r.choice(np.array([0.0, 0.2, 0.6, 1.0], np.float32), B)
    dt = r.choice(np.array([0.0, 0.5, 1.0], np.float32), B)
    x, d, tokens, u = make_drafts(r, B, N, V, dtype, scale, dt, 0.5)
    got = iw.drafts.verify_drafts(x.cuda(), tokens.cuda(), d.cuda(), T(u), temperature=T(t), scale=scale,
                                  draft_temperature=T(dt), draft_scale=scale * 0.9)
    check_verdict(got, x, tokens, d, u, None, t, scale, dt, scale * 0.9)
    got = iw.drafts.verify_drafts(x.cuda(), tokens.cuda(), d.cuda(), T(u), temperature=0.0, scale=scale, draft_temperature=1.0)
    check_verdict(got, x, tokens, d, u, None, 0.0, scale, 1.0)
    greedy = x.double().argmax(-1)
    for b in range(B):  # temperature 0 is greedy decoding whatever is drafted
        a = int(got.accepted[b])
        assert torch.equal(got.choice[b, :a + 1].cpu(), greedy[b, :a + 1])


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_verify_suppressed_and_outside(iw, gpu, dtype):
    """Suppressed drafts and drafts outside the vocabulary are refused, and never drawn."""
    print("case: verify suppressed", dtype, flush=True)
    r = gen.rng(6)
    B, N, V = 20, 4, 5001
    scale = 0.125 if dtype == "int8" else 1.0
    x, d, tokens, u = make_drafts(r, B, N, V, dtype, scale, 1.0, 0.3)
    off = sorted(set(r.integers(0, V, 40).tolist()) | set(x[:, 1].double().argmax(-1).tolist()))
    tokens[3, 1], tokens[4, 2], tokens[5, 1], tokens[6, 1] = V, -1, 2 ** 62, -2 ** 63
    tokens[7, 1] = off[3]
    for draft in (d, None):
        got = iw.drafts.verify_drafts(x.cuda(), tokens.cuda(), None if draft is None else draft.cuda(), T(u), scale=scale,
                                      suppress=T(bit_words(off, V)))
        check_verdict(got, x, tokens, draft, u, None, 1.0, scale, suppress=off)
        assert (got.accepted[[3, 5, 6, 7]] == 0).all() and int(got.accepted[4]) <= 1


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_verify_equal_distributions(iw, gpu, dtype):
    """Drafts of the model's own distribution are all accepted, whatever the numbers; a draft that it cannot have
    made leaves the model's distribution."""
    print("case: verify equal", dtype, flush=True)
    r = gen.rng(7)
    B, N, V = 16, 6, 2050
    scale = 0.125 if dtype == "int8" else 1.0
    x, _, _, u = make_drafts(r, B, N, V, dtype, scale, 1.0)
    d = x[:, :N - 1]
    tokens = torch.from_numpy(r.integers(0, V, (B, N)))
    u[0] = 1.0 - 2.0 ** -24
    got = iw.drafts.verify_drafts(x.cuda(), tokens.cuda(), d.cuda(), T(u), scale=scale)
    assert (got.accepted == N - 1).all()
    check_verdict(got, x, tokens, d, u, None, 1.0, scale)
    tokens[:, 1] = V  # no token: refused, and nothing is left of p - q
    got = iw.drafts.verify_drafts(x.cuda(), tokens.cuda(), d.cuda(), T(u), scale=scale)
    assert (got.accepted == 0).all()
    check_verdict(got, x, tokens, d, u, None, 1.0, scale)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_verify_special_values(iw, gpu, dtype):
    """Rows of NaN, of infinities, of masked logits on either side."""
    print("case: verify special", dtype, flush=True)
    r = gen.rng(8)
    B, N, V = 14, 4, 3001
    x, d, tokens, u = make_drafts(r, B, N, V, dtype, 1.0, 1.0, 0.2)
    x[0, 0, 7] = math.nan
    x[1, 1, 7] = math.inf
    x[2, 0] = -math.inf
    x[3, 3, 9] = math.nan
    d[4, 0, 9] = math.nan
    d[5, 1] = -math.inf
    d[6, 0, 1] = math.inf
    x[7, :, 100:] = -math.inf
    d[8, :, 100:] = -math.inf
    tokens[8, 1:] = 200
    x[9] = torch.finfo(x.dtype).min
    x[10, :, ::2] = torch.finfo(x.dtype).min
    u[11] = math.nan
    u[12], u[13] = -5.0, 7.0
    for draft in (d, None):
        got = iw.drafts.verify_drafts(x.cuda(), tokens.cuda(), None if draft is None else draft.cuda(), T(u))
        check_verdict(got, x, tokens, draft, u, None, 1.0, 1.0)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_verify_strides(iw, gpu, dtype):
    """Padded rows, drafts' logits node by node, rows at odd addresses."""
    print("case: verify strides", dtype, flush=True)
    r = gen.rng(9)
    B, N, V = 5, 4, 1003
    scale = 0.125 if dtype == "int8" else 1.0
    x, d, tokens, u = make_drafts(r, B, N, V, dtype, scale, 1.0)
    want = iw.drafts.verify_drafts(x.cuda(), tokens.cuda(), d.cuda(), T(u), scale=scale)
    check_verdict(want, x, tokens, d, u, None, 1.0, scale)
    wide = torch.full((B, N, V + 9), 90, dtype=x.dtype, device="cuda")
    wide[..., 3:3 + V] = x.cuda()
    nodes_first = d.transpose(0, 1).contiguous().cuda().transpose(0, 1)
    got = iw.drafts.verify_drafts(wide[..., 3:3 + V], tokens.cuda(), nodes_first, T(u), scale=scale)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    one = x[:1].cuda().expand(B, N, V)  # one text for all rows
    got = iw.drafts.verify_drafts(one, tokens.cuda(), d.cuda(), T(u), scale=scale)
    check_verdict(got, x[:1].expand(B, N, V), tokens, d, u, None, 1.0, scale)


def test_verify_keeps_the_distribution(iw, gpu):
    """Whatever the drafts are drawn from, the first token of a row is distributed as the model's: of 2^17 rows, within six
    deviations; and so is the second where the first was accepted."""
    print("case: verify distribution", flush=True)
    n, V, t = 1 << 17, 12, 0.9
    r = gen.rng(11)
    x = torch.from_numpy(r.normal(0, 1.5, (3, V))).float()
    d = torch.from_numpy(r.normal(0, 1.5, (2, V))).float()
    X, D = (a.cuda().expand(n, *a.shape) for a in (x, d))
    tokens = torch.zeros((n, 3), dtype=torch.int64, device="cuda")
    for i in range(2):
        tokens[:, i + 1] = iw.drafts.sample_tokens(D[:, i], T(r.random(n, np.float32)), temperature=t).tokens
    got = iw.drafts.verify_drafts(X, tokens, D, T(r.random((n, 3), np.float32)), temperature=t)
    p = torch.softmax(x.double() / t, 1).numpy()

    def close(tok, p):
        f = np.bincount(tok, minlength=V) / len(tok)
        assert (np.abs(f - p) <= 6 * np.sqrt(p * (1 - p) / len(tok))).all()
    choice, taken = host(got.choice), host(got.accepted)
    close(choice[:, 0], p[0])
    close(choice[taken >= 1, 1], p[1])
    close(choice[taken >= 2, 2], p[2])
    q = torch.softmax(d.double() / t, 1).numpy()
    rate = np.minimum(p[:2], q).sum(1)[0]  # of the first draft
    assert abs((taken >= 1).mean() - rate) <= 6 * math.sqrt(rate * (1 - rate) / n)


# ---------------------------------------------------------------------------
# streams, graphs, the whole loop
# ---------------------------------------------------------------------------

def test_captured_round_replays(iw, gpu):
    """A round of the three captured as one graph: every replay on new inputs, between eager rounds, gives the
    eager results."""
    print("case: captured round", flush=True)
    B, H, D, cap, N, V = 3, 2, 64, 300, 5, 20000
    C = H * D
    r = gen.rng(4)
    q, k, v = T(gen.i8(r, (B, N, C))), T(gen.i8(r, (B, H, cap, D))), T(gen.i8(r, (B, H, D, 304)))
    ln = T(np.array([300, 20, 150], np.int32))
    x, d, tokens, u = make_drafts(r, B, N, V, "int8", 0.125, 1.0)
    x, d, tokens, u = x.cuda(), d.cuda(), tokens.cuda(), T(u)
    un = T(r.random((B, N), np.float32))

    def round_():
        y = iw.drafts.window_attention(q, k, v, ln, heads=H, before=60, sinks=4, qk_multiplier=90, qk_shift=9, frac_bits=8,
                                       av_multiplier=100, av_shift=6)
        s = iw.drafts.sample_tokens(x, un, temperature=0.8, scale=0.125)
        return [y, *s, *iw.drafts.verify_drafts(x, tokens, d, u, temperature=0.8, scale=0.125)]
    round_()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = round_()
    for i in range(4):
        r = gen.rng(100 + i)
        q.copy_(T(gen.i8(r, (B, N, C))))
        ln.copy_(T(r.integers(0, cap + 1, B).astype(np.int32)))
        nx, nd, nt, nu = make_drafts(r, B, N, V, "int8", 0.125, 1.0)
        x.copy_(nx), d.copy_(nd), tokens.copy_(nt), u.copy_(T(nu))
        un.copy_(T(r.random((B, N), np.float32)))
        want = [a.clone() for a in round_()]
        for a in outs:
            a.fill_(77)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_two_streams_at_once(iw, gpu):
    """Calls with workspaces of their own, queued on two streams."""
    print("case: two streams", flush=True)
    r = gen.rng(5)
    cases = [make_drafts(gen.rng(i), 8, 4, 30000, "bfloat16", 1.0, 1.0) for i in range(2)]
    cases = [(x.cuda(), t.cuda(), d.cuda(), T(u)) for x, d, t, u in cases]
    wins = [Window(i, 2, 2, 128, 5000, 2, 3000, 0, 4, lengths=[5000, 4000 + i]) for i in range(2)]
    wargs = [(w, *w.args()) for w in wins]

    def both(i):
        w, a, o = wargs[i]
        return [*iw.drafts.verify_drafts(*cases[i]), *iw.drafts.sample_tokens(cases[i][0], cases[i][3]),
                iw.drafts.window_attention(*a, **o, **w.kw())]
    want = [both(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((i, both(i)))
    torch.cuda.synchronize()
    for i, out in got:
        assert all(torch.equal(a, b) for a, b in zip(out, want[i]))


def test_empty_batches(iw, gpu):
    print("case: empty", flush=True)
    z = torch.zeros
    i8 = dict(dtype=torch.int8, device="cuda")
    out = iw.drafts.window_attention(z((0, 3, 128), **i8), z((0, 2, 40, 64), **i8), z((0, 2, 64, 48), **i8), heads=2, before=4,
                                     qk_multiplier=1, qk_shift=1, frac_bits=8, av_multiplier=1, av_shift=1)
    assert out.shape == (0, 3, 128)
    out = iw.drafts.window_attention(z((2, 0, 128), **i8), z((2, 2, 40, 64), **i8), z((2, 2, 64, 48), **i8), heads=2, before=4,
                                     qk_multiplier=1, qk_shift=1, frac_bits=8, av_multiplier=1, av_shift=1)
    assert out.shape == (2, 0, 128)
    got = iw.drafts.sample_tokens(z((0, 100), device="cuda"), z(0, device="cuda"))
    assert got.tokens.shape == (0,)
    got = iw.drafts.sample_tokens(z((2, 0, 100), device="cuda"), z((2, 0), device="cuda"))
    assert got.tokens.shape == (2, 0)
    got = iw.drafts.verify_drafts(z((0, 3, 50), device="cuda"), z((0, 3), dtype=torch.int64, device="cuda"),
                                  z((0, 2, 50), device="cuda"), z((0, 3), device="cuda"))
    assert got.choice.shape == (0, 3) and got.accepted.shape == (0,)


def small_model(iw, heads=6, d=384, vocab=512, text_ctx=48):
    dims = iw.ModelDimensions(n_mels=80, n_audio_ctx=64, n_audio_state=d, n_audio_head=heads, n_audio_layer=2,
                              n_vocab=vocab, n_text_ctx=text_ctx, n_text_state=d, n_text_head=heads, n_text_layer=2)
    P = iw.synth.calibrated_int_params(dims, seed=11)
    return dims, iw.Whisper_int.from_params(dims, P).cuda()


PROMPT = np.array([[1, 2, 3], [4, 5, 6], [7, 8, 9]], np.int64)


def drafted(iw, model, dims, nodes, steps, t, seed=3, until=None, **kw):
    """A DraftDecoder's run: the rows' tokens, its steps, the decoder."""
    B = len(PROMPT)
    mel = iw.synth.synthetic_mel(B, dims.n_mels, 2 * dims.n_audio_ctx, seed=21)
    feats = model.embed_audio(T(mel))
    runner = iw.DecoderRunner(model.decoder, B, dims.n_audio_ctx)
    runner.set_audio(feats)
    dec = iw.drafts.DraftDecoder(runner, nodes, **kw)
    r = gen.rng(seed)
    last = dec.start(T(PROMPT), T(r.random(B, np.float32)), t)
    out = [[int(x)] for x in last]
    done = []
    while len(done) < steps and (until is None or min(map(len, out)) < until):
        frames = T(r.integers(0, dims.n_audio_ctx, B).astype(np.int32)) if kw.get("audio") is not None else None
        res = dec.step(last, T(r.random((B, 2 * nodes - 1), np.float32)), t, frames=frames)
        n = host(res.accept.accepted)
        for b in range(B):
            out[b] += host(res.verdict.choice)[b, :n[b]].tolist()
            if n[b]:
                assert out[b][-1] == int(res.accept.next_token[b])
        last = torch.where(res.accept.next_token >= 0, res.accept.next_token, last)
        done.append(res)
    return out, done, dec, feats


@pytest.mark.parametrize("heads", [6, 4])
@pytest.mark.parametrize("nodes,kw", [(1, {}), (4, {}), (5, dict(window=2, sinks=1)), (4, dict(window=0, sinks=0)),
                                      (6, dict(window=5, audio=3, audio_sinks=2))])
def test_draft_decoder_at_temperature_0(iw, gpu, heads, nodes, kw):
    """Greedy decoding's tokens, whatever window the drafts are made over."""
    print("case: draft decoder greedy", heads, nodes, kw, flush=True)
    dims, model = small_model(iw, heads=heads)
    with torch.no_grad():
        out, _, dec, feats = drafted(iw, model, dims, nodes, 60, 0.0, until=25, **kw)
        want = host(iw.greedy_decode(model, feats, T(PROMPT), 25))[:, 3:]
    assert [o[:25] for o in out] == want.tolist()


@pytest.mark.parametrize("heads", [6, 4])
def test_draft_decoder_that_sees_all(iw, gpu, heads):
    """Drafts made over all keys have the model's own distribution: every one is accepted, until the cache is full."""
    print("case: draft decoder sees all", heads, flush=True)
    dims, model = small_model(iw, heads=heads)
    with torch.no_grad():
        out, done, dec, _ = drafted(iw, model, dims, 5, 9, 1.0)
    for res in done[:8]:  # 3 + 8 * 5 of 48 positions
        assert (res.verdict.accepted == 4).all() and (res.accept.accepted == 5).all()
    assert torch.equal(done[8].accept.accepted.cpu(), torch.full((3,), 5, dtype=torch.int32))
    assert (dec.lengths == 48).all()


@pytest.mark.parametrize("heads", [6, 4])
def test_draft_decoder_caches(iw, gpu, heads):
    """Sampled with small windows: the caches are those of a decoder that was given the accepted tokens, and every
    step's tokens are what its logits and numbers say."""
    print("case: draft decoder caches", heads, flush=True)
    dims, model = small_model(iw, heads=heads)
    with torch.no_grad():
        out, done, dec, feats = drafted(iw, model, dims, 4, 8, 1.0, window=3, sinks=1)
        n = min(map(len, out)) - 1
        assert n >= 8
        forced = iw.DecoderRunner(model.decoder, 3, dims.n_audio_ctx)
        forced.set_audio(feats)
        forced.run_forced(T(PROMPT), T(np.array([o[:n] for o in out])))
        assert any((res.verdict.accepted < 3).any() for res in done)
        r = dec.runner
        for l in range(dims.n_text_layer):
            m = 3 + n
            assert torch.equal(r.k_self[l][:, :, :m], forced.k_self[l][:, :, :m])
            a, b = (x.v_self[l].view(dec.tree.v_cache[l].shape) for x in (r, forced))
            if r.v_quads:
                a, b = (x.transpose(3, 4).flatten(2, 3)[:, :, :m] for x in (a, b))
            else:
                a, b = a[..., :m], b[..., :m]
            assert torch.equal(a, b)


def test_draft_decoder_step_replays(iw, gpu):
    """A captured step: its replays on new numbers advance the rows as eager steps do."""
    print("case: draft decoder replays", flush=True)
    dims, model = small_model(iw)
    B, N, rounds = 3, 4, 6
    mel = iw.synth.synthetic_mel(B, dims.n_mels, 2 * dims.n_audio_ctx, seed=22)
    last = torch.zeros(B, dtype=torch.int64, device="cuda")
    u = torch.zeros((B, 2 * N - 1), device="cuda")
    frames = torch.zeros(B, dtype=torch.int32, device="cuda")
    with torch.no_grad():
        feats = model.embed_audio(T(mel))
        runs = []
        for captured in (False, True):
            runner = iw.DecoderRunner(model.decoder, B, dims.n_audio_ctx)
            runner.set_audio(feats)
            dec = iw.drafts.DraftDecoder(runner, N, window=4, audio=10, audio_sinks=2)
            r = gen.rng(9)
            if captured:
                dec.start(T(PROMPT), u[:, 0].contiguous())
                dec.step(last, u, frames=frames)
                torch.cuda.synchronize()
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g):
                    res = dec.step(last, u, frames=frames)
            last.copy_(dec.start(T(PROMPT), T(r.random(B, np.float32))))
            kept = []
            for _ in range(rounds):
                u.copy_(T(r.random((B, 2 * N - 1), np.float32)))
                frames.copy_(T(r.integers(0, 64, B).astype(np.int32)))
                if captured:
                    g.replay()
                else:
                    res = dec.step(last, u, frames=frames)
                last.copy_(res.accept.next_token)
                kept += [x.clone() for x in (res.tokens, *res.verdict, *res.accept, dec.lengths)]
                torch.cuda.synchronize()
            runs.append(kept)
        assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_draft_decoder_ends_at_eot(iw, gpu):
    """An accepted end-of-text ends the step's tokens; suppressed tokens never come up."""
    print("case: draft decoder eot", flush=True)
    dims, model = small_model(iw)
    with torch.no_grad():
        out, done, *_ = drafted(iw, model, dims, 4, 1, 1.0)
        eot = int(done[0].verdict.choice[0, 1])
        B = len(PROMPT)
        mel = iw.synth.synthetic_mel(B, dims.n_mels, 2 * dims.n_audio_ctx, seed=21)
        runner = iw.DecoderRunner(model.decoder, B, dims.n_audio_ctx)
        runner.set_audio(model.embed_audio(T(mel)))
        dec = iw.drafts.DraftDecoder(runner, 4)
        r = gen.rng(3)
        last = dec.start(T(PROMPT), T(r.random(B, np.float32)), 1.0)
        res = dec.step(last, T(r.random((B, 7), np.float32)), 1.0, eot=eot)
        assert int(res.accept.next_token[0]) == eot
        assert int(res.verdict.choice[0, int(res.accept.accepted[0]) - 1]) == eot
        even = T(bit_words(range(0, 512, 2), 512))
        out, *_ = drafted(iw, model, dims, 4, 4, 1.0, suppress=even)
    assert all(x % 2 == 1 for o in out for x in o)
