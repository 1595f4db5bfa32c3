"""Token scores at the ends of their ranges, against float64: scales and logits whose products or
distances leave float32, rows with NaN. Captured rounds and filled workspaces, compared to the byte."""
import numpy as np
import pytest
import torch

from tests import gen
from tests.test_speculative import Case, T, bit_words, host, logits_of, random_tree

FLOATS = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
FLT_MAX = float(np.finfo(np.float32).max)


def check(got, logits, targets, top, scale, suppress=()):
    """Against float64, with the tolerances of test_speculative.check_scores: 600 * 2^-24 for what an
    exp enters, three roundings of a log-probability itself. One that float32 does not reach is -inf."""
    x = logits.double().numpy().copy()
    x[:, list(suppress)] = -np.inf
    scale = float(np.float32(scale))
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        d = (x - x.max(1, keepdims=True)) * scale
        e = np.exp(d)
        lp = d - np.log(e.sum(1, keepdims=True))
        entropy = -np.where(e > 0, np.exp(lp) * lp, 0).sum(1)
    lp[lp < -FLT_MAX] = -np.inf
    r = 600 * 2.0 ** -24

    def close(a, b, room):
        a, fin = host(a).astype(np.float64), np.isfinite(b)
        assert np.array_equal(np.isneginf(a), np.isneginf(b)) and not np.isnan(a).any(), (a, b)
        assert (np.abs(a[fin] - b[fin]) <= room[fin]).all(), (a[fin], b[fin])

    def room(b):
        return r + np.where(np.isfinite(b), np.abs(b), 0) * 3 * 2.0 ** -24
    close(got.entropy, entropy, r * (1 + np.abs(entropy)))
    want = lp[np.arange(len(lp)), targets]
    close(got.logprob, want, room(want))
    ids = np.argsort(-x, axis=1, kind="stable")[:, :top]
    assert np.array_equal(host(got.top_ids), ids)
    want = np.take_along_axis(lp, ids, 1)
    close(got.top_logprobs, want, room(want))


@pytest.mark.gpu
@pytest.mark.parametrize("V", [300, 5000, 70001])
@pytest.mark.parametrize("dtype", list(FLOATS))
@pytest.mark.parametrize("scale", [2.0 ** -100, 2.0 ** -60, 1e-7, 2.4e7, 6e7, 1e8, 1.1e9, 1e10, 1e12, 1e20, 1e30, 2e38,
                                   3.3e38])
def test_masked_rows_under_any_scale(iw, gpu, scale, dtype, V):
    """-inf, suppressed tokens and the type's lowest value have no probability under small and large
    scales, beside logits that differ by about 1 / scale and by far more."""
    print("case: masked rows", scale, dtype, V, flush=True)
    r = gen.rng(V)
    x = logits_of(r, 5, V, "float32", 1.0)
    x[0] = torch.from_numpy(r.uniform(0, min(5 / scale, 3e38), V))
    x[1] = torch.from_numpy(r.uniform(-1, 0, V) * min(30 / scale, 3e38))
    x = x.clamp(torch.finfo(FLOATS[dtype]).min, torch.finfo(FLOATS[dtype]).max).to(FLOATS[dtype])
    x[:3, ::3] = -np.inf
    x[3, 1::2] = torch.finfo(x.dtype).min
    tg = np.array([1, 2, 0, 5, 7])
    got = iw.speculative.token_logprobs(x.cuda(), T(tg), top=4, scale=scale)
    check(got, x, tg, 4, scale)
    off = r.integers(0, V, 20)
    got = iw.speculative.token_logprobs(x.cuda(), T(tg), top=4, scale=scale, suppress=T(bit_words(off, V)))
    check(got, x, tg, 4, scale, off)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("scale", [2.0 ** -100, 2.0 ** -70, 1e-10, 0.5, 0.99, 1.0, 3.0])
def test_logits_further_apart_than_float32(iw, gpu, scale, dtype):
    """v - m passes float32 where (v - m) * scale need not."""
    print("case: far apart", scale, dtype, flush=True)
    r = gen.rng(5)
    x = torch.from_numpy(r.uniform(-3.3e38, 3.3e38, (6, 900))).to(FLOATS[dtype])
    x[:, 3], x[:, 4], x[4, 5] = 3.3e38, -3.3e38, -np.inf
    x[5] = torch.finfo(x.dtype).min
    x[5, 8] = torch.finfo(x.dtype).max
    tg = np.array([4, 4, 3, 700, 5, 8])
    check(iw.speculative.token_logprobs(x.cuda(), T(tg), top=32, scale=scale), x, tg, 32, scale)
    two = x[:, 3:5].contiguous()
    tg = np.array([0, 1, 1, 0, 1, 1])
    check(iw.speculative.token_logprobs(two.cuda(), T(tg), top=2, scale=scale), two, tg, 2, scale)
    long = torch.zeros((6, 70001), dtype=x.dtype)  # rows in parts
    long[:, -900:] = x
    long[:, 0] = -3.3e38
    tg = np.array([0, 69101 + 4, 69101 + 3, 5, 0, 69101])
    check(iw.speculative.token_logprobs(long.cuda(), T(tg), top=32, scale=scale), long, tg, 32, scale)


def nan_order(row, top):
    """Columns in the order of alternatives: NaN first, then by value, ties to the lowest index."""
    v = row.double().tolist()
    return sorted(range(len(v)), key=lambda i: (0, 0.0, i) if v[i] != v[i] else (1, -v[i], i))[:top]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(FLOATS))
@pytest.mark.parametrize("V,top", [(1, 1), (2, 2), (5, 5), (32, 32), (40, 7), (3000, 32), (51865, 3), (70001, 32)])
def test_alternatives_of_rows_with_nan(iw, gpu, V, top, dtype):
    """A NaN is the largest wherever it stands, the first column and whole rows included; as many
    alternatives as there are tokens are all of them."""
    print("case: nan order", V, top, dtype, flush=True)
    r = gen.rng(V)
    x = logits_of(r, 7, V, dtype, 1.0)
    x[0, 0] = np.nan
    x[1] = np.nan
    x[2, ::2] = np.nan
    x[3, V - 1] = -torch.tensor(np.nan)
    x[4], x[4, 0] = np.inf, np.nan
    x[5], x[5, 0] = -np.inf, np.nan
    x[6] = -np.inf
    tg = np.zeros(7, np.int64)
    got = iw.speculative.token_logprobs(x.cuda(), T(tg), top=top)
    assert host(got.top_ids).tolist() == [nan_order(row, top) for row in x]
    assert bool(got.logprob.isnan().all()) and bool(got.entropy.isnan().all())
    assert bool(got.top_logprobs.isnan().all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["int8", "float32"])
def test_as_many_rows_as_a_call_takes(iw, gpu, dtype):
    """2^22 rows: the scores of a row are those of the same row among few; one row more is refused."""
    print("case: 2^22 rows", dtype, flush=True)
    V, n = 3, 1 << 22
    few = T(gen.i8(gen.rng(1), (64, V), -40, 40)).to(getattr(torch, dtype))
    tg = torch.arange(64, device="cuda") % V
    want = iw.speculative.token_logprobs(few, tg, top=2, scale=0.1)
    got = iw.speculative.token_logprobs(few.repeat(n // 64, 1), tg.repeat(n // 64), top=2, scale=0.1)
    r = 600 * 2.0 ** -24
    assert torch.equal(got.top_ids, want.top_ids.repeat(n // 64, 1))
    for a, b in ((got.logprob, want.logprob.repeat(n // 64)), (got.entropy, want.entropy.repeat(n // 64)),
                 (got.top_logprobs, want.top_logprobs.repeat(n // 64, 1))):
        assert bool(((a - b).abs() <= r * (1 + b.abs())).all())
    with pytest.raises(RuntimeError, match="2\\^22 rows"):
        iw.speculative.token_logprobs(few[:1].repeat(n + 1, 1))


def differing(names, got, want):
    """Names of the outputs whose bytes are not the same."""
    return [n for n, a, b in zip(names, got, want, strict=True)
            if a.dtype != b.dtype or a.shape != b.shape
            or not torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))]


def test_differing_sees_one_byte():
    a = [torch.tensor([1, 2, 3]), torch.tensor([0.0, 1.0]), torch.tensor([float("nan")]), torch.zeros(2, 0)]
    names = "abcd"
    assert differing(names, a, [t.clone() for t in a]) == []
    for i, j, v in ((0, 2, 4), (1, 0, -0.0), (2, 0, 1.0)):
        b = [t.clone() for t in a]
        b[i][j] = v
        assert differing(names, b, a) == [names[i]]
    with pytest.raises(ValueError):
        differing(names, a[:3], a)


@pytest.mark.gpu
def test_captured_round_replays_byte_for_byte(iw, gpu):
    """Plan, attention, scores and acceptance captured as one graph: every replay on new inputs,
    between eager rounds of the same, leaves the eager outputs and caches to the byte."""
    sp = iw.speculative
    B, H, D, cap, N, V = 3, 2, 64, 96, 7, 70000
    C = H * D
    c = Case(1, B, H, D, cap, N, [10, 50, 80], [7, 5, 7], "quads")
    qkv, k, v = T(c.qkv), T(c.k), c.v_view(T(c.vc))
    ln, cnt, par = T(c.lengths), T(c.counts), T(c.parents)
    logits = T(gen.i8(gen.rng(3), (B, N, V)))
    tok, eot = torch.zeros((B, N), dtype=torch.int64, device="cuda"), 2
    caches = sp.TreeCaches([qkv[..., C:2 * C]], [qkv[..., 2 * C:]], [k], [v], heads=H)
    names = ("visible", "positions", "attention", "logprob", "entropy", "top_ids", "top_logprobs", "path", "accepted", "next",
             "lengths", "k", "v")

    def round_():
        plan = sp.tree_plan(par, cnt, lengths=ln, max_positions=cap)
        y = sp.tree_attention(qkv[..., :C], qkv[..., C:2 * C], qkv[..., 2 * C:], k, v, ln, plan.visible, cnt, heads=H,
                              qk_multiplier=90, qk_shift=9, frac_bits=8, av_multiplier=100, av_shift=6)
        s = sp.token_logprobs(logits, tok, top=3, scale=0.1)
        a = caches.accept(tok, par, s.top_ids[..., 0].contiguous(), ln, cnt, eot=eot)
        return [*plan, y, *s, *a]
    round_()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = round_()
    accepted = set()
    for i in range(6):
        r = gen.rng(100 + i)
        qkv.copy_(T(gen.i8(r, c.qkv.shape)))
        x = gen.i8(r, (B, N, V), -127, 100)
        top = r.integers(0, 3, (B, N))
        x[np.arange(B)[:, None], np.arange(N), top] = 127  # few choices, so that paths go on
        logits.copy_(T(x))
        par.copy_(T(random_tree(r, B, N)))
        ln.copy_(T(r.integers(0, cap - N, B).astype(np.int32)))
        cnt.copy_(T(r.integers(0, N + 1, B).astype(np.int32)))
        tok.copy_(T(r.integers(0, 3, (B, N))))
        saved = k.clone(), v.clone()
        want = [t.clone() for t in round_()] + [k.clone(), v.clone()]
        k.copy_(saved[0]), v.copy_(saved[1])
        g.replay()
        torch.cuda.synchronize()
        assert differing(names, [*outs, k, v], want) == []
        accepted |= set(host(outs[8]).tolist())
    assert len(accepted) > 2  # paths of several lengths


GUARD = 4096


def workspace(iw, name, sizes, fill):
    """A workspace of the size that the entry point names, filled, with a guard behind it."""
    need = iw._lib.value(name, *sizes)
    assert need > 0
    w = torch.full((need + GUARD,), fill, dtype=torch.uint8, device="cuda")
    return w, need


@pytest.mark.gpu
@pytest.mark.parametrize("fill", [0x00, 0x7f, 0xff])
@pytest.mark.parametrize("layout", ["vt", "quads"])
@pytest.mark.parametrize("D,cap,N", [(128, 1536, 1), (96, 1600, 16), (80, 2100, 17), (128, 2049, 33), (112, 1999, 64),
                                     (64, 8192, 5), (48, 8300, 50)])
def test_tree_attention_any_workspace(iw, oracle, gpu, D, cap, N, layout, fill):
    """Whatever the workspace holds before, the outputs are the same and nothing behind it is written:
    parts without a chunk, with the tree alone, rows without nodes or keys."""
    print("case: attention workspace", D, cap, N, layout, fill, flush=True)
    B, H = 6, 1
    c = Case(cap, B, H, D, cap, N, [0, 1, cap, cap // 2, 0, cap // 3], [N, 1, N, (N + 1) // 2, N, 0], layout)
    c.visible[4] = 0
    C = H * D
    w, need = workspace(iw, "iw_attention_tree_workspace", (B, H, N, D, cap), fill)
    qkv, k, vc, ln, vis, cnt = T(c.qkv), T(c.k), c.v_view(T(c.vc)), T(c.lengths), T(c.visible), T(c.counts)
    out = torch.full((B, N, C), 77, dtype=torch.int8, device="cuda")
    vs = vc.stride()
    v_s = (vs[0], vs[1], 4, vs[2]) if layout == "quads" else (vs[0], vs[1], vs[2], 4)
    qm, qs, f, am, as_ = c.sc
    q = qkv.data_ptr()
    args = iw.speculative._pack(iw.speculative._ATTENTION_ARGS, q, N * 3 * C, 3 * C, q + C, N * 3 * C, 3 * C, q + 2 * C,
                                N * 3 * C, 3 * C, k.data_ptr(), *k.stride()[:3], vc.data_ptr(), *v_s, ln.data_ptr(),
                                vis.data_ptr(), N, cnt.data_ptr(), out.data_ptr(), N * C, C, B, H, N, D, cap, qm, qs, f, am,
                                as_, 16, w.data_ptr())
    iw._lib.call("iw_attention_tree", args, iw._lib.stream())
    assert np.array_equal(host(out), c.expected(oracle))
    assert bool((w[need:] == fill).all())


@pytest.mark.gpu
@pytest.mark.parametrize("fill", [0x00, 0x7f, 0xff])
@pytest.mark.parametrize("kind,dtype", enumerate(["int8", "float32", "bfloat16", "float16"]))
@pytest.mark.parametrize("V,top", [(65537, 32), (70001, 0), (200003, 9)])
def test_token_logprobs_any_workspace(iw, gpu, V, top, kind, dtype, fill):
    print("case: scores workspace", V, top, dtype, fill, flush=True)
    r = gen.rng(V)
    scale = 0.125 if dtype == "int8" else 0.5
    x, tg = logits_of(r, 5, V, dtype, scale), r.integers(0, V, 5)
    x[1] = x[1].abs()
    if dtype != "int8":
        x[2, V // 2:] = -np.inf
    xd, t = x.cuda(), T(tg)
    w, need = workspace(iw, "iw_token_logprobs_workspace", (kind, 5, V, top), fill)
    lp, ent, lps = (torch.full(s, 7.0, device="cuda") for s in ((5,), (5,), (5, max(top, 1))))
    ids = torch.full((5, max(top, 1)), -7, dtype=torch.int64, device="cuda")
    iw._lib.call("iw_token_logprobs", xd.data_ptr(), kind, 5, V, V, scale, None, t.data_ptr(), lp.data_ptr(), ent.data_ptr(),
                 top, ids.data_ptr(), lps.data_ptr(), w.data_ptr(), iw._lib.stream())
    assert bool((w[need:] == fill).all())
    got = iw.speculative.TokenLogprobs(lp, ent, ids[:, :top], lps[:, :top])
    check(got, x, tg, top, scale)
