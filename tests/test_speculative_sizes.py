"""Drafted-token operators at layouts and sizes between and beyond those of test_speculative.py:
caches in other orders of their dims, the longest cache, rows of very many parts, a context that fills up."""
import numpy as np
import pytest
import torch

from tests import gen
from tests.test_speculative import Case, T, check_scores, host, logits_of, small_model, walk

pytestmark = pytest.mark.gpu


def reordered(x, *order):
    """The same values with the dims laid out in memory in this order."""
    back = [order.index(i) for i in range(len(order))]
    return x.permute(*order).contiguous().permute(*back)


@pytest.mark.parametrize("layout", ["vt", "quads"])
@pytest.mark.parametrize("cap,N", [(130, 5), (500, 33), (2100, 18)])
def test_caches_in_other_orders(iw, oracle, gpu, cap, N, layout):
    """Positions before heads, heads before rows: attention and acceptance as over the usual order."""
    print("case: cache orders", cap, N, layout, flush=True)
    sp = iw.speculative
    B, H, D = 3, 2, 96
    C = H * D
    c = Case(cap, B, H, D, cap, N, [0, cap // 2, cap - N], [N, N - 1, N], layout)
    want = c.expected(oracle)
    qm, qs, f, am, as_ = c.sc
    qkv, ln, vis, cnt, par = T(c.qkv), T(c.lengths), T(c.visible), T(c.counts), T(c.parents)
    tok = torch.zeros((B, N), dtype=torch.int64, device="cuda")
    plain = None
    for ko, vo in (((0, 1, 2, 3), (0, 1, 2, 3, 4)), ((0, 2, 1, 3), (0, 2, 1, 3, 4)), ((2, 0, 1, 3), (1, 2, 0, 3, 4)),
                   ((1, 0, 2, 3), (2, 1, 0, 3, 4))):
        k, v = reordered(T(c.k), *ko), c.v_view(T(c.vc))
        v = reordered(v, *vo) if layout == "quads" else reordered(v, *{0: (0, 1, 2, 3), 2: (0, 2, 1, 3)}.get(vo[1], (1, 2, 0, 3)))
        got = sp.tree_attention(qkv[..., :C], qkv[..., C:2 * C], qkv[..., 2 * C:], k, v, ln, vis, cnt, heads=H, qk_multiplier=qm,
                                qk_shift=qs, frac_bits=f, av_multiplier=am, av_shift=as_)
        assert np.array_equal(host(got), want)
        a = sp.TreeCaches([qkv[..., C:2 * C]], [qkv[..., 2 * C:]], [k], [v], heads=H).accept(tok, par, tok, ln, cnt)
        res = [*a, k, v]
        plain = plain or res
        assert all(torch.equal(x, y) for x, y in zip(res, plain))
    for b in range(B):
        path, _ = walk([0] * N, c.parents[b], [0] * N, c.counts[b], cap - c.lengths[b], -1)
        assert int(plain[1][b]) == len(path) > 0


@pytest.mark.parametrize("layout,cap", [("vt", (1 << 24) - 1), ("quads", 3_000_001)])
def test_longest_cache(iw, oracle, gpu, layout, cap):
    """All positions cached, up to 2^24 - 1."""
    print("case: longest cache", layout, cap, flush=True)
    c = Case(1, 1, 1, 16, cap, 2, [cap], [2], layout)
    assert np.array_equal(host(c.run(iw)), c.expected(oracle))


def test_operands_shared_by_rows(iw, oracle, gpu):
    """One row's projection expanded over the batch."""
    c = Case(8, 3, 2, 64, 100, 9, [0, 50, 100], [9, 9, 9], "quads")
    c.qkv[:] = c.qkv[:1]
    c.visible[:] = c.visible[:1]
    want = c.expected(oracle)
    one = T(c.qkv[:1]).expand(3, 9, 384)
    qm, qs, f, am, as_ = c.sc
    got = iw.speculative.tree_attention(one[..., :128], one[..., 128:256], one[..., 256:], T(c.k), c.v_view(T(c.vc)),
                                        T(c.lengths), T(c.visible[0]), heads=2, qk_multiplier=qm, qk_shift=qs, frac_bits=f,
                                        av_multiplier=am, av_shift=as_)
    assert np.array_equal(host(got), want)


@pytest.mark.parametrize("dtype,V", [("int8", (1 << 23) - 1), ("int8", 5_000_011), ("float32", 1_100_003),
                                     ("float32", (1 << 23) - 1), ("bfloat16", 2_200_001), ("float16", (1 << 23) - 1)])
@pytest.mark.parametrize("top", [0, 5, 32])
def test_rows_of_many_parts(iw, gpu, dtype, V, top):
    """More alternatives of the parts than the join holds at once; ties across parts."""
    print("case: many parts", dtype, V, top, flush=True)
    r = gen.rng(V)
    scale = 0.125 if dtype == "int8" else 1.0
    x = logits_of(r, 2, V, dtype, scale)
    x[1, :: V // 40] = x[1].max()
    tg = np.array([V - 1, V // 40])
    got = iw.speculative.token_logprobs(x.cuda(), T(tg), top=top, scale=scale)
    check_scores(got, x, tg, top, scale)


@pytest.mark.parametrize("heads", [6, 4])
@pytest.mark.parametrize("nodes", [1, 4, 16])
def test_tree_decoder_fills_the_context(iw, gpu, heads, nodes):
    """Chains of right drafts up to the last position: greedy_decode's tokens, one more that is not
    cached, then no room."""
    print("case: full context", heads, nodes, flush=True)
    dims, model = small_model(iw, heads=heads)
    B, P = 2, 3
    steps = dims.n_text_ctx - P
    mel = iw.synth.synthetic_mel(B, dims.n_mels, 2 * dims.n_audio_ctx, seed=23)
    prompt = T(np.array([[1, 2, 3], [4, 5, 6]], np.int64))
    with torch.no_grad():
        feats = model.embed_audio(T(mel))
        want = host(iw.greedy_decode(model, feats, prompt, steps))[:, P:]
        runner = iw.DecoderRunner(model.decoder, B, dims.n_audio_ctx)
        runner.set_audio(feats)
        tree = iw.speculative.TreeDecoder(runner, nodes)
        out = [[int(t)] for t in host(tree.start(prompt))]
        parents = torch.arange(-1, nodes - 1, dtype=torch.int32, device="cuda").repeat(B, 1)
        for _ in range(steps + 2):
            tokens = np.zeros((B, nodes), np.int64)
            for b in range(B):
                draft = want[b, len(out[b]) - 1:][:nodes]
                tokens[b, :len(draft)] = draft
            res = tree.step(T(tokens), parents)
            n, nxt, path = host(res.accept.accepted), host(res.accept.next_token), host(res.accept.path)
            for b in range(B):
                assert path[b, :n[b]].tolist() == list(range(n[b]))
                out[b] += [int(t) for t in tokens[b, 1:n[b]]] + ([int(nxt[b])] if n[b] else [])
                assert n[b] or (nxt[b] == -1 and int(tree.lengths[b]) == dims.n_text_ctx)
            if not n.any():
                break
        assert [o[:steps] for o in out] == want.tolist() and all(len(o) == steps + 1 for o in out)
        assert (host(tree.lengths) == dims.n_text_ctx).all()


@pytest.mark.parametrize("dtype", ["int8", "float32", "bfloat16", "float16"])
def test_suppressed_words_of_the_runners(iw, gpu, dtype):
    """The uint32 words of a runner's filters."""
    V = 5003
    r = gen.rng(3)
    x, off = logits_of(r, 3, V, dtype, 0.5), sorted(set(r.integers(0, V, 300).tolist()))
    words = np.zeros((V + 31) // 32, np.uint32)
    for i in off:
        words[i >> 5] |= np.uint32(1) << np.uint32(i & 31)
    tg = np.array([1, off[0], 2])
    got = iw.speculative.token_logprobs(x.cuda(), T(tg), top=6, scale=0.5, suppress=torch.from_numpy(words).cuda())
    check_scores(got, x, tg, 6, 0.5, off)


def test_tree_decoder_launches_on_its_device(iw, gpu, monkeypatch):
    """Every launch of a decoder's start and step is made with the tensors' device as the current
    one, whichever is current outside: of the calls into the library, those that name the stream of the
    current device are made within torch.cuda.device of the tensors'."""
    dims, model = small_model(iw)
    mel = iw.synth.synthetic_mel(1, dims.n_mels, 2 * dims.n_audio_ctx, seed=24)
    sp, entered, outside, streams = iw.speculative, [], [], []

    class Device(torch.cuda.device):
        def __enter__(self):
            entered.append(self.idx)
            return super().__enter__()

        def __exit__(self, *a):
            entered.pop()
            return super().__exit__(*a)
    with torch.no_grad():
        runner = iw.DecoderRunner(model.decoder, 1, dims.n_audio_ctx)
        runner.set_audio(model.embed_audio(T(mel)))
        tree = sp.TreeDecoder(runner, 3)
        call, launch = iw._lib.call, sp._launch
        own = []  # within _launch, which turns to the tensors' device itself

        def counted(name, *args):
            streams.append(name)
            if not own and entered[-1:] != [0]:
                outside.append(name)
            return call(name, *args)

        def launching(*args):
            own.append(1)
            try:
                return launch(*args)
            finally:
                own.pop()
        monkeypatch.setattr(torch.cuda, "device", Device)
        monkeypatch.setattr(iw._lib, "call", counted)
        monkeypatch.setattr(sp, "_launch", launching)
        last = tree.start(T(np.array([[1, 2, 3]], np.int64)))
        tokens = torch.cat([last, last, last])[None].contiguous()
        tree.step(tokens, torch.tensor([[-1, 0, 1]], dtype=torch.int32, device="cuda"))
        torch.cuda.synchronize()
    assert len(streams) > 20 and outside == []
