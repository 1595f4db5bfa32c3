"""The operators of sampled decoding at the ends of what they take: workspaces of any content, caches in
other orders, keys beyond 32-bit offsets, the widest vocabularies and the most rows, graphs on two streams,
a decoder on its device and in a graph."""
import numpy as np
import pytest
import torch

from tests import gen
from tests.test_drafts import DTYPES, T, Window, check_samples, check_verdict, host, make_drafts, make_logits, small_model
from tests.test_speculative_sizes import reordered

pytestmark = pytest.mark.gpu

GUARD = 4096


def workspace(iw, name, sizes, fill):
    """A workspace of the size that the entry point names, filled, with a guard behind it."""
    need = iw._lib.value(name, *sizes)
    assert need > 0
    return torch.full((need + GUARD,), fill, dtype=torch.uint8, device="cuda"), need


@pytest.mark.parametrize("fill", [0x00, 0x7f, 0xff])
@pytest.mark.parametrize("layout", ["vt", "quads"])
@pytest.mark.parametrize("D,cap,N,before", [(64, 9000, 1, 4500), (128, 20000, 1, 19000), (80, 6001, 1, 6000), (64, 9000, 2, 8000),
                                            (128, 5000, 17, 2500), (112, 4100, 33, 4099)])
def test_window_any_workspace(iw, oracle, gpu, D, cap, N, before, layout, fill):
    """Whatever the workspace holds before, the outputs are the same and nothing behind it is written: parts
    without a chunk, rows without queries or keys."""
    print("case: window workspace", D, cap, N, before, layout, fill, flush=True)
    B, H = 6, 1
    w = Window(cap + N, B, H, D, cap, N, before, 0, 40, lengths=[0, 1, cap, cap // 2, cap - 3, cap // 3],
               counts=[N, 1, N, (N + 1) // 2, N, 0], layout=layout)
    C = H * D
    work, need = workspace(iw, "iw_attention_window_workspace", (B, H, N, D, cap, before, 0, 40), fill)
    q, k, v, ln, cnt = T(w.q), T(w.k), w.v_view(T(w.vc)), T(w.lengths), T(w.counts)
    out = torch.full((B, N, C), 77, dtype=torch.int8, device="cuda")
    vs = v.stride()
    v_s = (vs[0], vs[1], 4, vs[2]) if layout == "quads" else (vs[0], vs[1], vs[2], 4)
    args = iw.drafts._pack(iw.drafts._WINDOW_ARGS, q.data_ptr(), N * 3 * C, 3 * C, k.data_ptr(), *k.stride()[:3], v.data_ptr(),
                           *v_s, ln.data_ptr(), 0, N, cnt.data_ptr(), out.data_ptr(), N * C, C, B, H, N, D, cap, before, 0, 40,
                           *w.sc, 16, work.data_ptr())
    iw._lib.call("iw_attention_window", args, iw._lib.stream())
    assert np.array_equal(host(out), w.expected(oracle))
    assert bool((work[need:] == fill).all())


@pytest.mark.parametrize("fill", [0x00, 0x7f, 0xff])
@pytest.mark.parametrize("kind,dtype", enumerate(DTYPES))
@pytest.mark.parametrize("V", [1, 4097, 70001])
def test_sampling_any_workspace(iw, gpu, V, kind, dtype, fill):
    print("case: sampling workspace", V, dtype, fill, flush=True)
    r = gen.rng(V)
    scale = 0.125 if dtype == "int8" else 1.0
    B, N = 3, 4
    x, d, tokens, u = make_drafts(r, B, N, V, dtype, scale, 0.9)
    counts = np.array([N, 2, 0], np.int32)
    xd, dd, td, ud, cd = x.cuda(), d.cuda(), tokens.cuda(), T(u), T(counts)
    work, need = workspace(iw, "iw_sample_tokens_workspace", (kind, B * N, V), fill)
    tok = torch.full((B * N,), -7, dtype=torch.int64, device="cuda")
    lp = torch.full((B * N,), 7.0, device="cuda")
    args = iw.drafts._pack(iw.drafts._SAMPLE_ARGS, xd.data_ptr(), kind, B * N, V, V, scale, 0.9, 0, 0, ud.data_ptr(),
                           tok.data_ptr(), lp.data_ptr(), work.data_ptr())
    iw._lib.call("iw_sample_tokens", args, iw._lib.stream())
    assert bool((work[need:] == fill).all())
    check_samples(iw.drafts.TokenSamples(tok, lp), x.reshape(B * N, V), u.reshape(-1), 0.9, scale)

    work, need = workspace(iw, "iw_verify_drafts_workspace", (kind, B, N, V, True), fill)
    choice = torch.full((B, N), -7, dtype=torch.int64, device="cuda")
    accepted = torch.full((B,), -7, dtype=torch.int32, device="cuda")
    nxt = torch.full((B,), -7, dtype=torch.int64, device="cuda")
    args = iw.drafts._pack(iw.drafts._VERIFY_ARGS, xd.data_ptr(), N * V, V, dd.data_ptr(), (N - 1) * V, V, kind, B, N, V, scale,
                           0.9, scale, 0.9, 0, 0, 0, td.data_ptr(), cd.data_ptr(), ud.data_ptr(), choice.data_ptr(),
                           accepted.data_ptr(), nxt.data_ptr(), work.data_ptr())
    iw._lib.call("iw_verify_drafts", args, iw._lib.stream())
    assert bool((work[need:] == fill).all())
    check_verdict(iw.drafts.DraftVerdict(choice, accepted, nxt), x, tokens, d, u, counts, 0.9, scale)


@pytest.mark.parametrize("layout", ["vt", "quads"])
@pytest.mark.parametrize("cap,N,before", [(130, 1, 64), (5000, 1, 4600), (500, 33, 100), (2100, 18, 2000)])
def test_window_caches_in_other_orders(iw, oracle, gpu, cap, N, before, layout):
    """Positions before heads, heads before rows; keys and values that rows of the batch share."""
    print("case: window cache orders", cap, N, layout, flush=True)
    B, H, D = 3, 2, 96
    w = Window(cap, B, H, D, cap, N, before, 0, 9, lengths=[cap, cap // 2, 3], layout=layout)
    want = w.expected(oracle)
    args, opt = w.args()
    for ko, vo in (((0, 2, 1, 3), (0, 2, 1, 3, 4)), ((2, 0, 1, 3), (1, 2, 0, 3, 4)), ((1, 0, 2, 3), (2, 1, 0, 3, 4))):
        k = reordered(args[1], *ko)
        v = reordered(args[2], *vo) if layout == "quads" else reordered(args[2], *((0, 2, 1, 3) if vo[1] == 2 else (1, 2, 0, 3)))
        got = iw.drafts.window_attention(args[0], k, v, args[3], **opt, **w.kw())
        assert np.array_equal(host(got), want)
    w.q[:], w.k[:], w.v[:], w.vc[:] = w.q[:1], w.k[:1], w.v[:1], w.vc[:1]
    args, opt = w.args()
    one = [a[:1].expand(B, *a.shape[1:]) for a in args[:3]]
    got = iw.drafts.window_attention(*one, args[3], **opt, **w.kw())
    assert np.array_equal(host(got), w.expected(oracle))


@pytest.mark.parametrize("layout", ["vt", "quads"])
@pytest.mark.parametrize("N", [1, 3, 40])
def test_window_far_keys(iw, oracle, gpu, N, layout):
    """Keys more than 2^32 bytes into a head of the longest cache, and heads as far apart."""
    print("case: window far keys", N, layout, flush=True)
    cap, D, near, H = (1 << 24) - 64, 128, 512, 2
    w = Window(N, 1, H, D, near, N, 200, 0, 16, lengths=[near], layout=layout)
    step = 512  # bytes of a key in the cache, of which a head has a quarter
    k = torch.zeros((cap, step), dtype=torch.int8, device="cuda")[:, :H * D].view(1, cap, H, D).transpose(1, 2)
    assert k.stride(2) * (cap - near) > 1 << 32
    k[:, :, -near:] = T(w.k)
    k[:, :, :16] = T(w.k)[:, :, :16]
    if layout == "vt":
        v = torch.zeros((1, H, D, cap), dtype=torch.int8, device="cuda")
        v[..., -near:] = T(w.v)
        v[..., :16] = T(w.v)[..., :16]
    else:
        v = torch.zeros((1, H, cap // 4, D, 4), dtype=torch.int8, device="cuda")
        v[:, :, -near // 4:] = w.v_view(T(w.vc))[:, :, :near // 4]
        v[:, :, :4] = w.v_view(T(w.vc))[:, :, :4]
    got = iw.drafts.window_attention(T(w.q)[..., :H * D], k, v, **w.kw())
    assert np.array_equal(host(got), w.expected(oracle))


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_sample_widest_vocabulary(iw, gpu, dtype):
    print("case: widest vocabulary", dtype, flush=True)
    V = (1 << 23) - 1
    r = gen.rng(3)
    scale = 0.125 if dtype == "int8" else 1.0
    x = make_logits(r, (2, V), dtype, scale)
    u = r.random(2, np.float32)
    check_samples(iw.drafts.sample_tokens(x.cuda(), T(u), scale=scale), x, u, 1.0, scale)


def test_sample_as_many_rows_as_a_call_takes(iw, gpu):
    """2^22 rows of two logits: which one is drawn follows from the number alone."""
    print("case: most rows", flush=True)
    n = 1 << 22
    x = torch.zeros((n, 2), dtype=torch.int8, device="cuda")
    x[1::2, 1] = 127
    u = (torch.arange(n, device="cuda") % 64).float() / 64
    got = iw.drafts.sample_tokens(x, u, temperature=0.01).tokens
    want = (u >= 0.5).long()
    want[1::2] = 1
    assert torch.equal(got, want)
    with pytest.raises(RuntimeError):
        iw.drafts.sample_tokens(torch.zeros((n + 1, 2), dtype=torch.int8, device="cuda"), torch.zeros(n + 1, device="cuda"))


def test_graphs_on_two_streams(iw, oracle, gpu):
    """Two captured calls with workspaces of their own, replayed on two streams at once."""
    print("case: graphs on two streams", flush=True)
    r = gen.rng(8)
    runs = []
    for i in range(2):
        w = Window(i, 2, 2, 128, 9000, 1 + 4 * i, 7000, 0, 4, lengths=[9000, 8000 + i], layout="quads")
        args, opt = w.args()
        x, d, tokens, u = make_drafts(r, 8, 4, 30000, "float16", 1.0, 1.0)
        x, d, tokens, u = x.cuda(), d.cuda(), tokens.cuda(), T(u)

        def run(w=w, args=args, opt=opt, x=x, d=d, tokens=tokens, u=u):
            return [iw.drafts.window_attention(*args, **opt, **w.kw()), *iw.drafts.sample_tokens(x, u),
                    *iw.drafts.verify_drafts(x, tokens, d, u)]
        want = [a.clone() for a in run()]
        assert np.array_equal(host(want[0]), w.expected(oracle))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = run()
        runs.append((g, outs, want, torch.cuda.Stream(), run))  # run holds the inputs
    torch.cuda.synchronize()
    for _ in range(5):
        for _, outs, *_ in runs:
            for a in outs:
                a.fill_(77)
        torch.cuda.synchronize()
        for g, _, _, s, _ in runs:
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for _, outs, want, *_ in runs:
            assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_draft_decoder_launches_on_its_device(iw, gpu, monkeypatch):
    """Every launch of a decoder's start and step is made with the tensors' device as the current
    one, whichever is current outside."""
    print("case: draft decoder's device", flush=True)
    dims, model = small_model(iw)
    mel = iw.synth.synthetic_mel(1, dims.n_mels, 2 * dims.n_audio_ctx, seed=24)
    entered, outside, streams, own = [], [], [], []

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
        dec = iw.drafts.DraftDecoder(runner, 3, window=2, audio=8)
        call, launch = iw._lib.call, iw.speculative._launch

        def counted(name, *args):
            streams.append(name)
            if not own and entered[-1:] != [0]:  # _launch turns to the tensors' device itself
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
        monkeypatch.setattr(iw.speculative, "_launch", launching)
        monkeypatch.setattr(iw.drafts, "_launch", launching)
        frames = torch.tensor([5], dtype=torch.int32, device="cuda")
        last = dec.start(T(np.array([[1, 2, 3]], np.int64)), torch.rand(1, device="cuda"))
        dec.step(last, torch.rand((1, 5), device="cuda"), frames=frames)
        torch.cuda.synchronize()
    assert {"iw_attention_window", "iw_sample_tokens", "iw_verify_drafts"} <= set(streams)
    assert outside == []


def test_draft_step_captured(iw, gpu):
    """A decoder's whole step as a graph: replays give what eager steps of a second decoder give."""
    print("case: captured step", flush=True)
    dims, model = small_model(iw)
    mel = T(iw.synth.synthetic_mel(2, dims.n_mels, 2 * dims.n_audio_ctx, seed=25))
    prompt = T(np.array([[1, 2, 3], [4, 5, 6]], np.int64))
    r = gen.rng(9)
    first, u = T(r.random(2, np.float32)), [T(r.random((2, 5), np.float32)) for _ in range(6)]
    with torch.no_grad():
        def decoder():
            runner = iw.DecoderRunner(model.decoder, 2, dims.n_audio_ctx)
            runner.set_audio(model.embed_audio(mel))
            dec = iw.drafts.DraftDecoder(runner, 3, window=4)
            return dec, dec.start(prompt, first, 0.9)
        dec, last = decoder()
        want = []
        for x in u:
            res = dec.step(last, x, 0.9)
            last = res.accept.next_token
            want.append([a.clone() for a in (*res.verdict, last, dec.lengths)])
        dec, last = decoder()
        now, x = last.clone(), u[0].clone()
        res = dec.step(now, x, 0.9)  # the first step, outside the graph
        got = [[a.clone() for a in (*res.verdict, res.accept.next_token, dec.lengths)]]
        now.copy_(res.accept.next_token)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = dec.step(now, x, 0.9)
        for i in range(1, len(u)):
            x.copy_(u[i])
            g.replay()
            torch.cuda.synchronize()
            got.append([a.clone() for a in (*res.verdict, res.accept.next_token, dec.lengths)])
            now.copy_(res.accept.next_token)
        for a, b in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))
