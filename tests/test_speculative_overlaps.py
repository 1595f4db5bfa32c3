"""Operands of the drafted-token operators that share memory: told apart exactly, refused where a
call would read what it writes. Grids beyond the launch limit. The refusals need no GPU."""
import random
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

from tests.test_speculative import Case, T, host
from tests.test_speculative_checks import ATTN, refused

CSRC = Path(__file__).resolve().parents[1] / "i-whisper_amd" / "csrc"
P = 1 << 30  # any address will do: a refused call reads nothing

DRIVER = r"""
#include <cstdio>
#include "iw_overlap.hpp"
using namespace iw;
int main() {
  char kind;
  while (std::scanf(" %c", &kind) == 1) {
    long long a[12];
    for (auto &x : a) std::scanf("%lld", &x);
    const auto at = [](long long x) { return reinterpret_cast<const void *>(x); };
    if (kind == 'r') {  // runs: at, bytes, stride, count of each
      std::printf("%d\n", (int)apart(Runs(at(a[0]), a[1], a[2], a[3]), Runs(at(a[4]), a[5], a[6], a[7])));
    } else {  // rows: batch, nodes, bytes, then base, sb, st of each
      const NodeRows x{at(a[3]), a[4], a[5], a[0], a[1], a[2]}, y{at(a[6]), a[7], a[8], a[0], a[1], a[2]};
      std::printf("%d %d\n", (int)apart(x, y), (int)rows_apart(x));
    }
  }
}
"""


@pytest.fixture(scope="module")
def overlap(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    d = tmp_path_factory.mktemp("overlap")
    (d / "driver.cpp").write_text(DRIVER)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Xlinker", "--no-undefined", f"-I{CSRC}", "driver.cpp", "-o", "driver"],
                   cwd=d, check=True)

    def run(lines):
        text = "\n".join(" ".join(map(str, [k, *v, *[0] * (12 - len(v))])) for k, v in lines)
        out = subprocess.run([d / "driver"], input=text, capture_output=True, text=True, check=True, timeout=60)
        return [tuple(map(int, x.split())) for x in out.stdout.splitlines()]
    return run


def touched(at, bytes_, *dims):
    """The bytes of runs at every combination of the (stride, count) dims."""
    starts = [at]
    for s, n in dims:
        starts = [x + s * i for x in starts for i in range(n)]
    return [x + j for x in starts for j in range(bytes_)]


def test_runs_are_told_apart(overlap):
    """Against sets of bytes: exact for runs of one stride, and never apart where a byte is shared."""
    r = random.Random(1)
    cases = []
    for _ in range(6000):
        same = r.random() < 0.7
        s = r.randint(-14, 14)
        a = [1000 + r.randint(-60, 60), r.randint(1, 9), s, r.randint(1, 6)]
        b = [1000 + r.randint(-60, 60), r.randint(1, 9), s if same else r.randint(-14, 14), r.randint(1, 6)]
        cases.append((a, b))
    got = overlap([("r", a + b) for a, b in cases])
    exact = 0
    for (a, b), (g,) in zip(cases, got, strict=True):
        want = not set(touched(a[0], a[1], a[2:])) & set(touched(b[0], b[1], b[2:]))
        assert not g or want, (a, b)
        if a[3] > 1 and b[3] > 1 and a[2] == b[2] != 0:
            assert g == want, (a, b)
            exact += 1
    assert exact > 1000


def test_rows_are_told_apart(overlap):
    r = random.Random(2)
    cases = []
    for _ in range(6000):
        batch, nodes, w = r.randint(1, 4), r.randint(1, 4), r.randint(1, 6)
        sb, st = r.randint(-40, 40), r.randint(-20, 20)
        x = [1000, sb, st]
        y = [1000 + r.randint(-80, 80), *((sb, st) if r.random() < 0.7 else (r.randint(-40, 40), r.randint(-20, 20)))]
        cases.append((batch, nodes, w, x, y))
    got = overlap([("n", [b, n, w, *x, *y]) for b, n, w, x, y in cases])
    exact = 0
    for (b, n, w, x, y), (g, own) in zip(cases, got, strict=True):
        bytes_ = touched(x[0], w, (x[1], b), (x[2], n))
        want = not set(bytes_) & set(touched(y[0], w, (y[1], b), (y[2], n)))
        assert not g or want, (b, n, w, x, y)
        assert own == (len(set(bytes_)) == len(bytes_)), (b, n, w, x)
        if x[1:] == y[1:] and 0 not in x[1:]:
            assert g == want, (b, n, w, x, y)
            exact += 1
    assert exact > 1000
    # addresses and strides near the ends of 64 bits
    far = (1 << 62) // 16 * 16
    assert overlap([("r", [far, 16, far, 2, 16, 16, far, 2]), ("n", [1 << 20, 64, 16, far, far, 1 << 40, 32, far, 1 << 40])])


# q, k_new, v_new, K and V of one row of 8 nodes and 2 heads of 64, 32 positions, without overlap
LAID = dict(ATTN, q=P, kn=P + 2048, vn=P + 4096, k=P + 8192, v=P + 16384, lengths=P + 24576, visible=P + 24640,
            out=P + 32768, batch=2, k_sb=4096, v_sb=4096)


@pytest.mark.parametrize("change,what", [
    (dict(o_st=0), "rows of out"), (dict(o_sb=0), "rows of out"), (dict(o_st=112), "rows of out"), (dict(o_sb=512), "rows of out"),
    (dict(out=P + 128), "overlap q"), (dict(out=P, o_st=256, o_sb=2048), "overlap q"), (dict(out=P, q_sb=2048), "overlap q"),
    (dict(out=P + 2048), "k_new"), (dict(out=P + 2048 - 16), "overlap q"), (dict(out=P + 4096 - 16), "k_new"),
    (dict(out=P + 6144 - 16), "k_new or v_new"), (dict(out=P + 4096), "k_new or v_new"),
    (dict(q=P, q_sb=4096, q_st=512, kn=P + 128, kn_sb=4096, kn_st=512, vn=P + 256, vn_sb=4096, vn_st=512, out=P + 16, o_sb=4096,
          o_st=512), "overlap q"),
    (dict(q=P, q_sb=4096, q_st=512, kn=P + 128, kn_sb=4096, kn_st=512, vn=P + 256, vn_sb=4096, vn_st=512, out=P + 240, o_sb=4096,
          o_st=512), "k_new"),
    (dict(out=P + 8192), "caches"), (dict(out=P + 8192 - 2032, o_sb=1024), "caches"), (dict(out=P + 16384 - 16), "caches"),
    (dict(out=P + 16384 + 4096), "caches"), (dict(out=P + 24576 - 16), "caches"),
    (dict(v_sq=4, v_sd=32, out=P + 16384 + 2 * 4096 - 16), "caches")])
def test_attention_refuses_shared_memory(iw, change, what):
    refused(iw, "iw_attention_tree", {**LAID, **change}, {}, what)


@pytest.mark.gpu
@pytest.mark.parametrize("N,cap", [(5, 130), (33, 130), (64, 500), (40, 4096)])
def test_out_in_the_place_of_q_and_between_columns(iw, oracle, gpu, N, cap):
    """out may be q itself, other columns of the projection's rows, or rows between those of the nodes."""
    print("case: out beside q", N, cap, flush=True)
    H, D = 2, 96
    C = H * D
    c = Case(N, 3, H, D, cap, N, [0, cap // 2, cap], [N, N - 1, N], "quads")
    want = c.expected(oracle)
    qm, qs, f, am, as_ = c.sc
    k, v, ln, vis, cnt = T(c.k), c.v_view(T(c.vc)), T(c.lengths), T(c.visible), T(c.counts)
    x = torch.zeros((N, 3, 5 * C), dtype=torch.int8, device="cuda").transpose(0, 1)  # the nodes' rows outermost
    y = torch.zeros((3, N, 5 * C), dtype=torch.int8, device="cuda")
    for buf in (x, y):
        for lo in (0, 3 * C, 4 * C):
            buf.fill_(55)
            buf[..., :3 * C] = T(c.qkv)
            out = buf[..., lo:lo + C]
            got = iw.speculative.tree_attention(buf[..., :C], buf[..., C:2 * C], buf[..., 2 * C:3 * C], k, v, ln, vis, cnt,
                                                heads=H, qk_multiplier=qm, qk_shift=qs, frac_bits=f, av_multiplier=am,
                                                av_shift=as_, out=out)
            assert got.data_ptr() == out.data_ptr() and np.array_equal(host(got), want)
            assert np.array_equal(host(buf[..., C:3 * C]), c.qkv[..., C:])
            other = [i for i in (3 * C, 4 * C) if i != lo]
            assert all(bool((buf[..., i:i + C] == 55).all()) for i in other)
    sc = dict(heads=H, qk_multiplier=qm, qk_shift=qs, frac_bits=f, av_multiplier=am, av_shift=as_)
    for lo in (16, C - 16, C, 2 * C, 3 * C - 16):
        with pytest.raises(RuntimeError, match="overlap"):
            iw.speculative.tree_attention(y[..., :C], y[..., C:2 * C], y[..., 2 * C:3 * C], k, v, ln, vis, cnt,
                                          out=y[..., lo:lo + C], **sc)
    for cache in (k, v):
        with pytest.raises(RuntimeError, match="caches"):
            iw.speculative.tree_attention(y[..., :C], y[..., C:2 * C], y[..., 2 * C:3 * C], k, v, ln, vis, cnt,
                                          out=cache.flatten()[-3 * N * C:].view(3, N, C), **sc)


def buf(*shape):
    return torch.zeros(shape, dtype=torch.int8)


def test_written_tensors_have_memory_of_their_own(iw):
    """Parts of one buffer in any order of its dims are told apart from those that share a byte."""
    own = iw.speculative._own_memory
    x = buf(3, 4, 2, 5, 8)  # [batch, layers, K or V, positions, D]
    parts = [x[:, l, i] for l in range(4) for i in range(2)]
    assert own(parts, []) and own(parts[:4], parts[4:]) and own([], parts + parts) and own([], [])
    assert own(parts[:3], [parts[3], parts[3]])
    assert not own(parts + parts[:1], []) and not own(parts, parts[:1])
    assert not own([x[:, 0], x[:, 0, 1]], []) and not own([x[:, 0, 0]], [x[2, 0, 0, 4, 7:]])
    assert own([x[:, 0, 0]], [x[2, 0, 1, 0, :1]])
    assert own([x[..., :4], x[..., 4:]], []) and not own([x[..., :5], x[..., 4:]], [])
    assert own([x.transpose(0, 3)], []) and own([x[:, :, :, ::2], x[:, :, :, 1::2]], [])
    assert not own([x[:1].expand(3, 4, 2, 5, 8)], [])
    flat = buf(1000)
    assert not own([flat.as_strided((4, 10), (9, 1))], []) and own([flat.as_strided((4, 10), (10, 1))], [])
    assert not own([flat[:500], flat[499:]], []) and own([flat[:500], flat[500:]], [])
    assert not own([flat[:500]], [flat[499:]]) and own([flat[:500]], [flat[500:]])
    assert own([buf(0, 4), buf(0, 4), flat[:0]], [buf(0)])
    assert own([flat[10:20], flat[30:40]], [flat[20:30], flat[:10], flat[40:]])
    assert not own([flat[10:20], flat[30:40]], [flat[25:31]]) and not own([flat[10:20], flat[30:40]], [flat[19:22]])


def test_written_tensors_against_sets_of_bytes(iw):
    own = iw.speculative._own_memory
    r = random.Random(3)
    flat = buf(4000)
    seen = [0, 0]
    for _ in range(1500):
        def view():
            if r.random() < 0.5:  # a part of a padded block
                s = (96, 24, 4)
                shape = (r.randint(1, 3), r.randint(1, 4), r.randint(1, 4))
            else:
                s = tuple(r.choice((1, 2, 4, 12, 24, 96)) for _ in range(3))
                shape = tuple(r.randint(0 if r.random() < 0.05 else 1, 4) for _ in range(3))
            return flat.as_strided(shape, s, r.randint(0, 200))
        written, read = [view() for _ in range(r.randint(0, 3))], [view() for _ in range(r.randint(0, 2))]

        def bytes_of(t):
            return touched(t.data_ptr(), 1, *zip(t.stride(), t.shape))
        w = [b for t in written for b in bytes_of(t)]
        want = len(set(w)) == len(w) and not set(w) & {b for t in read for b in bytes_of(t)}
        assert own(written, read) == want, [(t.stride(), t.shape, t.storage_offset()) for t in written + read]
        seen[want] += bool(w)
    assert min(seen) > 200


@pytest.mark.gpu
def test_tree_caches_memory(iw, gpu):
    """Caches that are parts of one buffer accept as separate ones do; ones that share memory are refused."""
    sp = iw.speculative
    L, B, H, T_, D, N = 3, 2, 2, 32, 64, 4
    C = H * D
    qkv = [torch.randint(-127, 128, (B, N, 3 * C), dtype=torch.int8, device="cuda") for _ in range(L)]
    kn, vn = [x[..., C:2 * C] for x in qkv], [x[..., 2 * C:] for x in qkv]
    one = torch.zeros((B, L, 2, H, T_ * D), dtype=torch.int8, device="cuda")
    k = [one[:, l, 0].unflatten(2, (T_, D)) for l in range(L)]
    v = [one[:, l, 1].unflatten(2, (T_ // 4, D, 4)) for l in range(L)]
    k2, v2 = [x.contiguous() for x in k], [x.contiguous() for x in v]
    tok = torch.zeros((B, N), dtype=torch.int64, device="cuda")
    par = torch.arange(-1, N - 1, dtype=torch.int32, device="cuda").repeat(B, 1)
    ln = torch.tensor([5, 31], dtype=torch.int32, device="cuda")
    a = sp.TreeCaches(kn, vn, k, v, heads=H).accept(tok, par, tok, ln)
    b = sp.TreeCaches(kn, vn, k2, v2, heads=H).accept(tok, par, tok, ln)
    assert host(a.accepted).tolist() == host(b.accepted).tolist() == [4, 1]
    assert all(torch.equal(x, y) for x, y in zip(k + v, k2 + v2)) and any(bool(x.any()) for x in k)
    near = torch.zeros(2 * B * H * T_ * D, dtype=torch.int8, device="cuda")
    k0 = near[:B * H * T_ * D].view(B, H, T_, D)
    for bad in ((kn, vn, k, k), (kn, vn, [k2[0], k2[0], k2[1]], v2)):
        with pytest.raises(RuntimeError, match="memory of its own|v_cache"):
            sp.TreeCaches(*bad, heads=H)
    with pytest.raises(RuntimeError, match="memory of its own"):
        sp.TreeCaches(kn[:1], vn[:1], [k0], [near[64:64 + k0.numel()].view(B, H, T_ // 4, D, 4)], heads=H)
    with pytest.raises(RuntimeError, match="memory of its own"):
        sp.TreeCaches([near[:3 * B * N * C].view(B, N, 3 * C)[..., :C]], vn[:1], [k0], v2[:1], heads=H)


@pytest.mark.gpu
def test_tree_caches_without_rows(iw, gpu):
    sp = iw.speculative
    e = lambda *shape, dtype=torch.int8: torch.empty(shape, dtype=dtype, device="cuda")
    caches = sp.TreeCaches([e(0, 4, 128)] * 2, [e(0, 4, 128)] * 2, [e(0, 2, 32, 64) for _ in range(2)],
                           [e(0, 2, 8, 64, 4) for _ in range(2)], heads=2)
    got = caches.accept(e(0, 4, dtype=torch.int64), e(0, 4, dtype=torch.int32), e(0, 4, dtype=torch.int64),
                        e(0, dtype=torch.int32))
    assert got.path.shape == (0, 4) and got.accepted.shape == got.next_token.shape == got.lengths.shape == (0,)


def test_grid_of_the_largest_batches(iw):
    """2^22 heads of 33 to 64 nodes over long caches would be 2^32 threads: refused by name."""
    far = 1 << 40
    big = dict(ATTN, q=far, kn=2 * far, vn=3 * far, k=4 * far, v=5 * far, lengths=6 * far, visible=7 * far, out=8 * far,
               batch=1 << 22, heads=1, nodes=64, D=16, cap=512, q_sb=1024, q_st=16, kn_sb=1024, kn_st=16, vn_sb=1024, vn_st=16,
               k_sb=8192, k_sh=8192, k_st=16, v_sb=8192, v_sh=8192, v_sd=4, v_sq=64, o_sb=1024, o_st=16)
    for nodes in (33, 64):
        refused(iw, "iw_attention_tree", big, dict(nodes=nodes), "too many heads")
    refused(iw, "iw_attention_tree", big, dict(batch=(1 << 22) - 3), "too many heads")


def test_addresses_are_compared_on_the_host(iw):
    """Whatever torch's default device is."""
    x = buf(2, 2, 8)
    with torch.device("meta"):
        assert iw.speculative._own_memory([x[:, 0], x[:, 1]], []) and not iw.speculative._own_memory([x[:, 0], x[:, 0]], [])
