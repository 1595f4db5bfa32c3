"""Drafted-token operators on the GPU against plain implementations.

* tree_attention: bit-exact with the CPU oracle's attention, row by row over the
  row's own keys and mask (all tile borders, both V layouts, ragged lengths and
  counts, empty rows, wrapping row maxima, every frac_bits)
* tree_plan, TreeCaches.accept: equal to walks on the host
* token_logprobs: float64 log-softmax, entropy and ordering on the host
* TreeDecoder: the tokens and caches of greedy_decode, whatever is drafted
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

def random_tree(r, B, N):
    """Parents of random trees, chains among them."""
    p = np.full((B, N), -1, np.int32)
    for b in range(B):
        for i in range(1, N):
            p[b, i] = i - 1 if b % 2 else max(0, i - 1 - int(r.integers(0, 4)))
    return p


def words(parents, counts):
    """The visibility words, by walking every node's path (as signed 64-bit)."""
    B, N = parents.shape
    out = np.zeros((B, N), np.uint64)
    for b in range(B):
        for i in range(counts[b]):
            j = i
            while 0 <= j <= i:
                out[b, i] |= np.uint64(1) << np.uint64(j)
                up = parents[b, j]
                j = up if up < j else -1
    return out.view(np.int64)


class Case:
    """Random operands with the caches' unused positions filled with noise."""

    def __init__(self, seed, B, H, D, cap, N, lengths, counts, layout, scalars=None, visible=None):
        r = gen.rng(seed)
        self.B, self.H, self.D, self.cap, self.N, self.layout = B, H, D, cap, N, layout
        C = H * D
        _, _, _, qm, qs, f, am, as_ = gen.attn_case(seed, 1, 1, 1, 1, D)
        self.sc = scalars or (qm, qs, f, am, as_)
        self.qkv = gen.i8(r, (B, N, 3 * C), -127, 127)
        self.k = gen.i8(r, (B, H, cap, D), -127, 127)
        self.v = gen.i8(r, (B, H, D, cap), -127, 127)
        self.lengths = np.asarray(lengths, np.int32)
        self.counts = np.asarray(counts, np.int32)
        self.parents = random_tree(r, B, N)
        self.visible = words(self.parents, self.counts) if visible is None else visible
        shape, self.vs = gen.v_cache_layout(B, H, D, cap, layout)
        self.vc = gen.i8(r, shape)
        gen.v_cache_put(self.vc, layout, 0, self.v)

    def v_view(self, vc):
        B, H, D = self.B, self.H, self.D
        if self.layout == "vt":
            return vc
        nq = vc.shape[2]
        return vc[..., :4 * D].unflatten(3, (D, 4)) if vc.shape[3] > 4 * D else vc.view(B, H, nq, D, 4)

    def run(self, iw, counts=True, **kw):
        C = self.H * self.D
        qkv = T(self.qkv)
        qm, qs, f, am, as_ = self.sc
        return iw.speculative.tree_attention(
            qkv[..., :C], qkv[..., C:2 * C], qkv[..., 2 * C:], T(self.k), self.v_view(T(self.vc)), T(self.lengths),
            T(self.visible), T(self.counts) if counts else None, heads=self.H, qk_multiplier=qm, qk_shift=qs,
            frac_bits=f, av_multiplier=am, av_shift=as_, **kw)

    def expected(self, oracle, rows=None):
        B, H, D, N, C = self.B, self.H, self.D, self.N, self.H * self.D
        out = np.zeros((B, N, C), np.int8)
        for b in range(B) if rows is None else rows:
            ln = min(max(int(self.lengths[b]), 0), self.cap)
            cnt = min(max(int(self.counts[b]), 0), N)
            if cnt == 0:
                continue
            q, kn, vn = (self.qkv[b, :cnt, i * C:(i + 1) * C].reshape(cnt, H, D).transpose(1, 0, 2) for i in range(3))
            k = np.concatenate([self.k[b, :, :ln], kn], 1)[None]
            v = np.concatenate([self.v[b, :, :, :ln], vn.transpose(0, 2, 1)], 2)[None]
            bits = (self.visible.reshape(-1, N)[b % self.visible.reshape(-1, N).shape[0], :cnt].view(np.uint64)[:, None]
                    >> np.arange(cnt, dtype=np.uint64)) & np.uint64(1)
            hidden = np.concatenate([np.zeros((cnt, ln), bool), bits == 0], 1)
            y = oracle.attention(np.ascontiguousarray(q[None]), k, v, hidden, *self.sc)[0]
            y[hidden.all(1)] = 0
            out[b, :cnt] = y
        return out


LAYOUTS = ("vt", "quads", "quads_pad")


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("N", [1, 2, 5, 15, 16, 17, 31, 32, 33, 47, 48, 49, 63, 64])
def test_tree_attention_nodes(iw, oracle, gpu, N, layout):
    print("case: tree attention nodes", N, layout, flush=True)
    c = Case(7 * N + 1, 3, 2, 64, 130, N, [0, 77, 130], [N, max(1, N - 1), (N + 1) // 2], layout)
    assert np.array_equal(host(c.run(iw)), c.expected(oracle))


@pytest.mark.parametrize("layout", ["vt", "quads"])
@pytest.mark.parametrize("D", [16, 32, 48, 64, 80, 96, 112, 128])
def test_tree_attention_head_dims(iw, oracle, gpu, D, layout):
    print("case: tree attention head dim", D, layout, flush=True)
    c = Case(D, 2, 3, D, 200, 21, [200, 101], [21, 20], layout)
    assert np.array_equal(host(c.run(iw)), c.expected(oracle))


@pytest.mark.parametrize("layout", ["vt", "quads"])
@pytest.mark.parametrize("length", [0, 1, 2, 3, 4, 5, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257, 447, 448])
def test_tree_attention_lengths(iw, oracle, gpu, length, layout):
    """Key counts that end inside a quad, a product, a chunk or the cache."""
    print("case: tree attention length", length, layout, flush=True)
    c = Case(3 * length + 2, 2, 4, 64, 448, 6, [length, 448 - length], [6, 4], layout)
    assert np.array_equal(host(c.run(iw)), c.expected(oracle))


@pytest.mark.parametrize("cap,D,N,layout", [(1, 64, 3, "vt"), (1, 64, 3, "quads"), (2, 128, 64, "quads"),
                                            (1500, 64, 9, "vt"), (4096, 64, 40, "quads"), (4095, 128, 61, "vt"),
                                            (9001, 32, 2, "quads")])
def test_tree_attention_caches(iw, oracle, gpu, cap, D, N, layout):
    print("case: tree attention cache", cap, D, N, layout, flush=True)
    c = Case(cap + D, 2, 2, D, cap, N, [cap, cap // 2 + 1], [N, N], layout)
    assert np.array_equal(host(c.run(iw)), c.expected(oracle))


@pytest.mark.parametrize("layout", ["vt", "quads"])
@pytest.mark.parametrize("B,H,D,cap,N", [(1, 20, 64, 100, 7), (40, 20, 64, 100, 7), (129, 3, 64, 100, 7),
                                         (65, 9, 64, 448, 33), (90, 6, 96, 448, 20), (300, 1, 64, 460, 3),
                                         (60, 9, 64, 500, 18), (60, 9, 128, 500, 18), (1, 1, 64, 100000, 2),
                                         (70, 10, 64, 130, 64), (70, 10, 96, 130, 61), (100, 10, 64, 500, 33),
                                         (100, 10, 128, 500, 40)])
def test_tree_attention_grids(iw, oracle, gpu, B, H, D, cap, N, layout):
    """Few and many blocks, one and two tiles of nodes a block, caches above 448 positions with
    their keys in one block and shared by several."""
    print("case: tree attention grid", B, H, D, cap, N, layout, flush=True)
    r = gen.rng(B)
    c = Case(B + H, B, H, D, cap, N, r.integers(0, cap + 1, B), r.integers(0, N + 1, B), layout)
    c.lengths[0], c.counts[0] = cap, N
    c.visible = words(c.parents, c.counts)
    rows = sorted({0, B - 1, *r.integers(0, B, 12).tolist()})
    assert np.array_equal(host(c.run(iw))[rows], c.expected(oracle, rows)[rows])


@pytest.mark.parametrize("layout", ["vt", "quads"])
@pytest.mark.parametrize("D,cap,N", [(128, 1536, 1), (128, 1600, 16), (80, 2100, 17), (128, 2049, 33), (112, 1999, 64),
                                     (64, 8192, 5), (48, 8300, 50)])
def test_tree_attention_shared_keys(iw, oracle, gpu, D, cap, N, layout):
    """Caches whose keys several blocks share: parts without a chunk, with the tree alone, rows without
    nodes or keys, and a workspace with other values in it."""
    print("case: tree attention shared keys", D, cap, N, layout, flush=True)
    B, H = 8, 1
    assert iw._lib.value("iw_attention_tree_workspace", B, H, N, D, cap) > 0
    c = Case(cap, B, H, D, cap, N, [0, 1, 64, cap - 1, cap, cap // 2, 0, cap // 3], [N, N, 1, N, N, (N + 1) // 2, N, 0], layout)
    c.visible[6] = 0  # no key at all
    c.visible[5, 0] = 0
    torch.full((1 << 23,), 0x7f, dtype=torch.uint8, device="cuda")
    want = c.expected(oracle)
    assert not want[6:].any()
    out = torch.full((B, N, H * D), 77, dtype=torch.int8, device="cuda")
    assert np.array_equal(host(c.run(iw, out=out)), want)
    assert np.array_equal(host(c.run(iw)), want)


@pytest.mark.parametrize("f", [1, 8, 10, 11, 13])
@pytest.mark.parametrize("qk", [(255, 0), (200, 4), (255, 40)])
def test_tree_attention_shared_keys_scalars(iw, oracle, gpu, f, qk):
    print("case: tree attention shared keys, scalars", f, qk, flush=True)
    c = Case(f, 2, 1, 96, 1700, 18, [1700, 900], [18, 11], "quads", scalars=(*qk, f, 255, 7))
    assert np.array_equal(host(c.run(iw)), c.expected(oracle))


@pytest.mark.parametrize("f", range(1, 14))
@pytest.mark.parametrize("qk", [(255, 0), (1, 0), (200, 4), (3, 9), (255, 31), (255, 40), (0, 3)])
def test_tree_attention_scalars(iw, oracle, gpu, f, qk):
    """Every frac_bits with scores that saturate (a row maximum of 32767 wraps),
    spread over the whole 16 bits, or all requantise to 0."""
    print("case: tree attention scalars", f, qk, flush=True)
    c = Case(f, 2, 2, 64, 150, 18, [150, 90], [18, 11], "quads", scalars=(*qk, f, 255, 7))
    assert np.array_equal(host(c.run(iw)), c.expected(oracle))


@pytest.mark.parametrize("av", [(255, 0), (1, 0), (130, 9), (255, 32), (255, -3)])
def test_tree_attention_output_scalars(iw, oracle, gpu, av):
    print("case: tree attention output scalars", av, flush=True)
    c = Case(5, 2, 2, 64, 60, 5, [60, 0], [5, 5], "vt", scalars=(90, 9, 8, *av))
    assert np.array_equal(host(c.run(iw)), c.expected(oracle))


@pytest.mark.parametrize("N", [5, 64])
def test_tree_attention_any_words(iw, oracle, gpu, N):
    """Words that are no tree's: nodes that see later nodes, unused ones or none at all."""
    print("case: tree attention words", N, flush=True)
    vis = gen.rng(N).integers(-2 ** 63, 2 ** 63, (3, N))
    vis[:, 1] = 0
    vis[:, 2] = -1
    c = Case(N, 3, 2, 64, 40, N, [0, 40, 0], [N, N - 1, 2], "quads", visible=vis)
    exp = c.expected(oracle)
    assert np.array_equal(host(c.run(iw)), exp)
    assert not exp[0, 1].any()  # no key seen


def test_tree_attention_shared_tree(iw, oracle, gpu):
    vis = words(random_tree(gen.rng(1), 1, 9), [9])[0]
    c = Case(2, 4, 2, 64, 40, 9, [40, 3, 0, 12], [9] * 4, "quads", visible=vis)
    assert np.array_equal(host(c.run(iw)), c.expected(oracle))
    assert np.array_equal(host(c.run(iw, counts=False)), c.expected(oracle))


def test_tree_attention_clamps_lengths_and_counts(iw, oracle, gpu):
    c = Case(3, 4, 2, 64, 70, 6, [-5, 10_000, 70, 2 ** 31 - 1], [6, 99, -1, 6], "quads",
             visible=np.full((4, 6), -1, np.int64))
    assert np.array_equal(host(c.run(iw)), c.expected(oracle))


def test_tree_attention_unused_nodes_are_zeros(iw, oracle, gpu):
    c = Case(4, 3, 2, 64, 70, 20, [5, 60, 70], [0, 3, 17], "vt")
    out = torch.full((3, 20, 256), 99, dtype=torch.int8, device="cuda")
    got = c.run(iw, out=out[..., :128])
    assert got.data_ptr() == out.data_ptr()
    assert np.array_equal(host(got), c.expected(oracle))
    assert bool((out[..., 128:] == 99).all())  # nothing beside the rows


def test_tree_attention_far_offsets(iw, oracle, gpu):
    """Rows of a cache more than 2^32 bytes apart."""
    c = Case(6, 2, 2, 64, 100, 5, [100, 37], [5, 5], "quads")
    far = 2 ** 32 + 4096
    size = 2 * 100 * 64
    k = torch.zeros(far + size, dtype=torch.int8, device="cuda")
    v = torch.zeros(far + 2 * 112 * 64, dtype=torch.int8, device="cuda")
    kv, vv = k.as_strided((2, 2, 100, 64), (far, 6400, 64, 1)), v.as_strided((2, 2, 28, 64, 4), (far, 7168, 256, 4, 1))
    kv.copy_(T(c.k))
    vv.copy_(c.v_view(T(c.vc)))
    C, qkv = 128, T(c.qkv)
    qm, qs, f, am, as_ = c.sc
    got = iw.speculative.tree_attention(qkv[..., :C], qkv[..., C:2 * C], qkv[..., 2 * C:], kv, vv, T(c.lengths),
                                        T(c.visible), heads=2, qk_multiplier=qm, qk_shift=qs, frac_bits=f,
                                        av_multiplier=am, av_shift=as_)
    assert np.array_equal(host(got), c.expected(oracle))


def test_tree_attention_equals_decode_attention(iw, gpu):
    """One node a row whose K and V are already the last cached ones' copies gives what
    iw_attention_decode_cache gives over length + 1 keys."""
    B, H, D, cap, n = 5, 4, 64, 448, 123
    c = Case(9, B, H, D, cap, 1, [n] * B, [1] * B, "quads")
    got = c.run(iw)
    C = H * D
    k, vc = T(c.k), T(c.vc)
    k[:, :, n] = T(c.qkv[:, 0, C:2 * C].reshape(B, H, D))
    vv = c.v_view(vc)
    vv[:, :, n // 4, :, n % 4] = T(c.qkv[:, 0, 2 * C:].reshape(B, H, D))
    q = T(np.ascontiguousarray(c.qkv[:, 0, :C]))
    out = torch.empty((B, C), dtype=torch.int8, device="cuda")
    qm, qs, f, am, as_ = c.sc
    iw._lib.call("iw_attention_decode_cache", q.data_ptr(), C, k.data_ptr(), H * cap * D, cap * D, D, vc.data_ptr(),
                 *c.vs, out.data_ptr(), C, B, H, D, n + 1, None, n + 1, qm, qs, f, am, as_, 16, iw._lib.stream())
    assert torch.equal(got[:, 0], out)


def test_tree_attention_refuses_layouts(iw, gpu):
    c = Case(1, 2, 2, 64, 33, 4, [3, 3], [4, 4], "vt")
    C, qkv = 128, T(c.qkv)
    sc = dict(heads=2, qk_multiplier=3, qk_shift=4, frac_bits=8, av_multiplier=3, av_shift=4)
    q, kn, vn = qkv[..., :C], qkv[..., C:2 * C], qkv[..., 2 * C:]
    k, v, ln, vis = T(c.k), T(c.vc), T(c.lengths), T(c.visible)
    f = iw.speculative.tree_attention
    assert f(q, kn, vn, k, v, ln, vis, **sc).shape == (2, 4, C)
    for bad, what in [((q.float(), kn, vn, k, v, ln, vis), "int8"), ((q, kn[:, :3], vn, k, v, ln, vis), "shape"),
                      ((q, kn, vn, k[:, :1], v, ln, vis), "shape"), ((q, kn, vn, k, v[..., :32], ln, vis), "round"),
                      ((q, kn, vn, k, v.transpose(2, 3), ln, vis), "shape"),
                      ((q, kn, vn, k.transpose(2, 3).contiguous().transpose(2, 3), v, ln, vis), "contiguous"),
                      ((q, kn, vn, k, v, ln.long(), vis), "int32"), ((q, kn, vn, k, v, ln[:1], vis), "shape"),
                      ((q, kn, vn, k, v, ln, vis.int()), "int64"), ((q, kn, vn, k, v, ln, vis[:, :3]), "shape"),
                      ((q, kn, vn, k, T(np.zeros((2, 2, 8, 64, 4), np.int8)), ln, vis), "every position"),
                      ((q.cpu(), kn, vn, k, v, ln, vis), "GPU|device"),
                      ((q, kn, vn, k, v, ln.cpu(), vis), "GPU"), ((q, kn, vn, k.cpu(), v, ln, vis), "GPU"),
                      ((q, kn, vn, k, v, None, vis), "tensor"), ((q, kn, vn, k, v, ln, None), "tensor")]:
        with pytest.raises(RuntimeError, match=what):
            f(*bad, **sc)
    with pytest.raises(RuntimeError, match="16-byte"):
        f(qkv[..., 1:C + 1], kn, vn, k, v, ln, vis, **sc)
    with pytest.raises(RuntimeError, match="overlap"):
        f(q, kn, vn, k, v, ln, vis, out=torch.empty(8 * C, dtype=torch.int8, device="cuda").as_strided((2, 4, C), (C, C, 1)), **sc)
    with pytest.raises(RuntimeError, match="overlap"):
        f(q, kn, vn, k, v, ln, vis, out=torch.empty(C, dtype=torch.int8, device="cuda").expand(2, 4, C), **sc)


# ---------------------------------------------------------------------------
# plan and acceptance
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("B,N", [(1, 1), (1, 8), (3, 33), (5, 64), (130, 64)])
def test_tree_plan(iw, gpu, B, N):
    print("case: tree plan", B, N, flush=True)
    r = gen.rng(B * N)
    p, cnt, ln = random_tree(r, B, N), r.integers(0, N + 1, B), r.integers(0, 448, B)
    p[0, N // 2] = N  # no earlier node: a root
    vis = words(p, cnt)
    pos = ln[:, None] + np.array([[max(0, bin(int(w) & (2 ** 64 - 1)).count("1") - 1) for w in row] for row in vis])
    got = iw.speculative.tree_plan(T(p), T(cnt.astype(np.int32)), lengths=T(ln.astype(np.int32)), max_positions=440)
    assert np.array_equal(host(got.visible), vis)
    assert np.array_equal(host(got.positions), np.minimum(pos, 439))
    got = iw.speculative.tree_plan(T(p))
    assert np.array_equal(host(got.visible), words(p, [N] * B))


def walk(tokens, parents, choice, cnt, room, eot):
    path = [0] if cnt > 0 and room > 0 else []
    while path and len(path) < room and not (eot >= 0 and choice[path[-1]] == eot):
        nxt = [j for j in range(path[-1] + 1, cnt) if parents[j] == path[-1] and tokens[j] == choice[path[-1]]]
        if not nxt:
            break
        path.append(nxt[0])
    return path, (choice[path[-1]] if path else -1)


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("L,B,H,D,cap,N", [(1, 1, 2, 64, 40, 1), (2, 3, 4, 64, 61, 12), (3, 7, 2, 96, 33, 64),
                                           (65, 2, 2, 16, 48, 9), (1, 2, 3, 128, 7, 20)])
def test_tree_accept(iw, gpu, L, B, H, D, cap, N, layout):
    """Few token values, so that paths are long and siblings hold the same token."""
    print("case: tree accept", L, B, H, D, cap, N, layout, flush=True)
    r = gen.rng(L + B + N)
    C = H * D
    tokens, choice = r.integers(0, 3, (B, N)), r.integers(0, 3, (B, N))
    parents = random_tree(r, B, N)
    counts, lengths = r.integers(0, N + 1, B), r.integers(0, cap + 1, B)
    counts[0], lengths[0] = N, max(0, cap - N)
    shape, _ = gen.v_cache_layout(B, H, D, cap, layout)
    qkv = [gen.i8(r, (B, N, 3 * C)) for _ in range(L)]
    ks, vs = [gen.i8(r, (B, H, cap, D)) for _ in range(L)], [gen.i8(r, shape) for _ in range(L)]
    q_d, k_d, v_d = [T(x) for x in qkv], [T(x) for x in ks], [T(x) for x in vs]

    def view(v):
        if layout == "vt":
            return v
        return v[..., :4 * D].unflatten(3, (D, 4)) if layout == "quads_pad" else v.view(B, H, -1, D, 4)
    caches = iw.speculative.TreeCaches([x[..., C:2 * C] for x in q_d], [x[..., 2 * C:] for x in q_d], k_d,
                                       [view(v) for v in v_d], heads=H)
    for eot in (-1, 2):
        got = caches.accept(T(tokens), T(parents), T(choice), T(lengths.astype(np.int32)), T(counts.astype(np.int32)),
                            eot=eot)
        path = np.full((B, N), -1, np.int32)
        for b in range(B):
            p, nxt = walk(tokens[b], parents[b], choice[b], counts[b], cap - lengths[b], eot)
            path[b, :len(p)] = p
            assert int(got.accepted[b]) == len(p) and int(got.next_token[b]) == nxt
            assert int(got.lengths[b]) == lengths[b] + len(p)
            for i, node in enumerate(p):
                at = lengths[b] + i
                for l in range(L):
                    ks[l][b, :, at] = qkv[l][b, node, C:2 * C].reshape(H, D)
                    gen.v_cache_put(vs[l][b:b + 1], layout, at, qkv[l][b, node, 2 * C:].reshape(1, H, D, 1))
        assert np.array_equal(host(got.path), path)
        for l in range(L):  # the path's positions and no other byte
            assert np.array_equal(host(k_d[l]), ks[l]) and np.array_equal(host(v_d[l]), vs[l])


def test_tree_caches_refuse(iw, gpu):
    f = iw.speculative.TreeCaches
    qkv = torch.zeros((2, 4, 3 * 128), dtype=torch.int8, device="cuda")
    kn, vn = qkv[..., 128:256], qkv[..., 256:]
    k = torch.zeros((2, 2, 32, 64), dtype=torch.int8, device="cuda")
    v = torch.zeros((2, 2, 8, 64, 4), dtype=torch.int8, device="cuda")
    f([kn], [vn], [k], [v], heads=2)
    with pytest.raises(RuntimeError, match="same strides"):
        f([kn, kn.contiguous()], [vn, vn], [k, k.clone()], [v, v.clone()], heads=2)
    with pytest.raises(RuntimeError, match="memory of its own"):
        f([kn, kn], [vn, vn], [k, k], [v, v.clone()], heads=2)
    with pytest.raises(RuntimeError, match="memory of its own"):
        f([kn], [vn], [k[:1].expand(2, 2, 32, 64)], [v], heads=2)
    with pytest.raises(RuntimeError, match="every position"):
        f([kn], [vn], [k], [v[:, :, :7]], heads=2)
    c = f([kn], [vn], [k], [v], heads=2)
    t, p, ln = (torch.zeros(s, dtype=d, device="cuda") for s, d in
                [((2, 4), torch.int64), ((2, 4), torch.int32), ((2,), torch.int32)])
    with pytest.raises(RuntimeError, match="int64"):
        c.accept(t.int(), p, t, ln)
    with pytest.raises(RuntimeError, match="shape"):
        c.accept(t[:, :3], p, t, ln)
    with pytest.raises(RuntimeError, match="shape"):
        c.accept(t, p, t, ln[:1])
    for eot in (1 << 63, 1 << 64, -(1 << 70)):
        with pytest.raises(RuntimeError, match="eot"):
            c.accept(t, p, t, ln, eot=eot)


# ---------------------------------------------------------------------------
# token scores
# ---------------------------------------------------------------------------

DTYPES = {"int8": torch.int8, "float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def logits_of(r, rows, V, dtype, scale):
    x = r.normal(-4, 2, (rows, V))
    for i in range(rows):
        x[i, r.integers(0, V, min(5, V))] += r.uniform(3, 20, min(5, V))
    t = torch.from_numpy(x / scale)
    if dtype == "int8":
        return t.round().clamp(-127, 127).to(torch.int8)
    return t.to(DTYPES[dtype])


def bit_words(ids, V):
    w = np.zeros((V + 31) // 32, np.uint32)
    for i in ids:
        w[i >> 5] |= np.uint32(1) << np.uint32(i & 31)
    return w.view(np.int32)


def check_scores(got, logits, targets, top, scale, suppress=()):
    """Against float64. With d = (x - m) scale, m the row maximum, down to -104 (below it exp is 0 in
    float32): d has two roundings and its product with log2 e a third, so exp(d) is off by at most
    3 * 104 * 2^-24 plus the instruction's 2^-23, and a sum of a thread's up to 128 terms, 64 lanes,
    16 waves and up to 128 blocks by 128 + 6 + 16 + 128 more roundings: r = 600 * 2^-24 relative covers
    Z' and U'. log1p(Z') is then off by at most r, a log-probability by r + 3 roundings of itself, the entropy by
    r (1 + H)."""
    x = logits.double().numpy().copy()
    x[:, list(suppress)] = -np.inf
    m = x.max(1, keepdims=True)
    with np.errstate(invalid="ignore", divide="ignore"):
        d = (x - m) * scale
        e = np.exp(d)
        lse = np.log(e.sum(1, keepdims=True))
        lp = d - lse
        H = -np.where(e > 0, np.exp(lp) * lp, 0).sum(1)
    r = 600 * 2.0 ** -24

    def close(a, b, room):
        a = a.double().cpu().numpy()
        assert np.array_equal(np.isinf(a), np.isinf(b))
        fin = np.isfinite(b)
        worst = np.abs(a[fin] - b[fin]) - room[fin]
        assert not worst.size or worst.max() <= 0, worst.max()
    close(got.entropy, H, r * (1 + np.abs(H)))
    if targets is not None:
        want = lp[np.arange(len(lp)), targets]
        close(got.logprob, want, r + np.where(np.isfinite(want), np.abs(want), 0) * 3 * 2.0 ** -24)
    if top:
        ids = np.argsort(-x, axis=1, kind="stable")[:, :top]
        assert np.array_equal(host(got.top_ids), ids)
        want = np.take_along_axis(lp, ids, 1)
        close(got.top_logprobs, want, r + np.where(np.isfinite(want), np.abs(want), 0) * 3 * 2.0 ** -24)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,V,top", [(1, 1, 1), (2, 2, 2), (3, 31, 5), (5, 33, 32), (2, 1000, 1), (4, 1025, 7),
                                        (3, 4099, 0), (2, 51865, 5), (300, 700, 3), (2, 65536, 4), (2, 65537, 32),
                                        (3, 200003, 9)])
def test_token_logprobs(iw, gpu, rows, V, top, dtype):
    print("case: token logprobs", rows, V, top, dtype, flush=True)
    r = gen.rng(rows + V + top)
    scale = 0.125 if dtype == "int8" else 0.5
    x = logits_of(r, rows, V, dtype, scale)
    tg = r.integers(0, V, rows)
    got = iw.speculative.token_logprobs(x.cuda(), T(tg), top=top, scale=scale)
    check_scores(got, x, tg, top, scale)
    off = r.integers(0, V, min(V - 1, V // 10 + 3)) if V > top + 40 else []
    got = iw.speculative.token_logprobs(x.cuda(), T(tg), top=top, scale=scale, suppress=T(bit_words(off, V)))
    check_scores(got, x, tg, top, scale, off)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("shift", [0, 1, 3, 7, 15])
def test_token_logprobs_strides(iw, gpu, shift, dtype):
    """Rows that start at any multiple of the type's size, apart by more than their length, whose
    neighbours hold larger values; leading dimensions."""
    print("case: token logprobs strides", shift, dtype, flush=True)
    r = gen.rng(shift)
    V = 4001
    wide = logits_of(r, 6, V + 30, dtype, 0.25)
    wide[:, :shift] = 127
    wide[:, shift + V:] = 127
    x = wide[:, shift:shift + V]
    got = iw.speculative.token_logprobs(wide.cuda()[:, shift:shift + V], top=3, scale=0.25)
    check_scores(got, x, None, 3, 0.25)
    cube = iw.speculative.token_logprobs(wide.cuda()[:, shift:shift + V].reshape(2, 3, V), top=3, scale=0.25)
    assert cube.top_ids.shape == (2, 3, 3) and cube.entropy.shape == (2, 3)
    assert torch.equal(cube.top_ids.view(6, 3), got.top_ids)
    one = iw.speculative.token_logprobs(x[0].contiguous().cuda(), torch.tensor(5, device="cuda"), top=2, scale=0.25)
    assert one.entropy.shape == () and one.logprob.shape == () and torch.equal(one.top_ids, got.top_ids[0, :2])


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("V", [5, 3000, 51865, 70001])
def test_token_logprobs_ties(iw, gpu, V, dtype):
    """Constant rows, rows of two values and ascending neighbours: ties go to the lowest index."""
    r = gen.rng(V)
    top = min(32, V)
    x = torch.zeros((5, V), dtype=torch.float32)
    x[1] = torch.from_numpy(r.integers(0, 2, V).astype(np.float32))
    x[2, V // 2:] = 3.0
    x[3] = torch.arange(V) % 100
    x[4, min(V - 1, 1000):min(V, 1040)] = 7.0
    x = x.to(DTYPES[dtype])
    got = iw.speculative.token_logprobs(x.cuda(), T(np.arange(5) % V), top=top)
    check_scores(got, x, np.arange(5) % V, top, 1.0)


@pytest.mark.parametrize("V", [300, 51865, 70001])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_token_logprobs_special_values(iw, gpu, V, dtype):
    """Masked tokens (-inf and the type's lowest value), zeros of both signs, NaN, +inf, empty rows."""
    print("case: token logprobs special", V, dtype, flush=True)
    r = gen.rng(V)
    x = logits_of(r, 8, V, dtype, 1.0)
    x[0, ::2] = -math.inf
    x[1, 1:] = -math.inf
    x[2, : V - 2] = torch.finfo(x.dtype).min
    x[3] = -math.inf
    x[4, V // 3] = math.nan
    x[5, V // 3] = math.inf
    x[6] = 0.0
    x[6, 1::2] = -0.0
    tg = np.array([1, 0, V - 1, 0, 5, 5, 3, 9])
    got = iw.speculative.token_logprobs(x.cuda(), T(tg), top=5)
    ok = [0, 1, 2, 6, 7]
    pick = type(got)(*[t[ok] for t in got])
    check_scores(pick, x[ok], tg[ok], 5, 1.0)
    for i in (3, 4, 5):  # no probabilities
        assert bool(got.logprob[i].isnan()) and bool(got.entropy[i].isnan()) and bool(got.top_logprobs[i].isnan().all())
    assert host(got.top_ids[3]).tolist() == [0, 1, 2, 3, 4]
    assert int(got.top_ids[4, 0]) == V // 3 and int(got.top_ids[5, 0]) == V // 3
    assert host(got.top_ids[6]).tolist() == [0, 1, 2, 3, 4]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("scale", [0.1, 0.3, 0.7, 1.1, 1.3, 2.0, 3.7])
def test_token_logprobs_scales_of_masked_rows(iw, gpu, scale, dtype):
    """-inf stays without probability under every scale, whatever the sign of its rounding."""
    r = gen.rng(int(10 * scale))
    x = logits_of(r, 4, 5000, dtype, 1.0)
    x[:, ::3] = -math.inf
    got = iw.speculative.token_logprobs(x.cuda(), T(np.array([1, 2, 0, 5])), top=4, scale=scale)
    check_scores(got, x, np.array([1, 2, 0, 5]), 4, float(np.float32(scale)))


@pytest.mark.parametrize("scale,size", [(2.0 ** -100, 2.0 ** 101), (2.0 ** -100, 3e38),
                                        (2.0 ** 120, 2.0 ** -118), (2e38, 1.0)])
def test_token_logprobs_extreme_scales(iw, gpu, scale, size):
    """Scales and logits near the ends of float32 (smaller scales are refused)."""
    r = gen.rng(7)
    x = torch.from_numpy(r.uniform(-1, 1, (3, 2000)) * size).float()
    got = iw.speculative.token_logprobs(x.cuda(), T(np.array([1, 2, 3])), top=2, scale=scale)
    with np.errstate(over="ignore"):
        lp = (x.double() * float(np.float32(scale))).log_softmax(1)
    want = lp[torch.arange(3), torch.tensor([1, 2, 3])]
    a = got.logprob.double().cpu()
    assert bool(((a - want).abs() <= 600 * 2.0 ** -24 + want.abs() * 2.0 ** -22).logical_or(
        (a == -math.inf) & (want < -3e38)).all())
    assert torch.equal(got.top_ids.cpu(), x.topk(2, 1).indices)


def test_token_logprobs_targets_outside(iw, gpu):
    x = torch.randn(4, 100)
    got = iw.speculative.token_logprobs(x.cuda(), T(np.array([-1, 100, 2 ** 40, 7])))
    assert host(got.logprob.isnan()).tolist() == [True, True, True, False]
    assert got.top_ids is None and got.top_logprobs is None


def test_token_logprobs_suppressed(iw, gpu):
    """Suppressed targets have no probability; a row without any other token has no scores;
    alternatives past the allowed ones are the suppressed ones in order."""
    V = 70
    x = torch.zeros((2, V), dtype=torch.int8)
    x[:, 3] = 50
    got = iw.speculative.token_logprobs(x.cuda(), T(np.array([3, 69])), top=4, suppress=T(bit_words(range(69), V)))
    assert float(got.logprob[0]) == -math.inf and float(got.logprob[1]) == 0.0 and float(got.entropy[1]) == 0.0
    assert host(got.top_ids).tolist() == [[69, 0, 1, 2]] * 2
    assert host(got.top_logprobs).tolist() == [[0.0] + [-math.inf] * 3] * 2
    got = iw.speculative.token_logprobs(x.cuda(), T(np.array([3, 4])), top=2, suppress=T(bit_words(range(70), V)))
    assert bool(got.logprob.isnan().all()) and bool(got.entropy.isnan().all())
    assert host(got.top_ids).tolist() == [[0, 1]] * 2


def test_token_logprobs_certain_rows(iw, gpu):
    """Log-probabilities and entropies far below 2^-24 keep their digits."""
    x = torch.full((2, 1000), -40.0)
    x[:, 17] = 0.0
    x[1, 18] = -20.0
    got = iw.speculative.token_logprobs(x.cuda(), T(np.array([17, 17])), top=1)
    z = np.array([999 * math.exp(-40.0), 998 * math.exp(-40.0) + math.exp(-20.0)])
    u = np.array([999 * 40 * math.exp(-40.0), 998 * 40 * math.exp(-40.0) + 20 * math.exp(-20.0)])
    assert np.allclose(host(got.logprob), -np.log1p(z), rtol=600 * 2.0 ** -24, atol=0)
    assert np.allclose(host(got.entropy), np.log1p(z) + u / (1 + z), rtol=600 * 2.0 ** -24, atol=0)


@pytest.mark.parametrize("dtype", ["int8", "bfloat16"])
def test_token_logprobs_far_rows(iw, gpu, dtype):
    """Rows and columns beyond 2^31 elements are those of a copy near the start."""
    print("case: far rows", dtype, flush=True)
    rows, V = 33000, 70001
    x = torch.empty((rows, V), dtype=DTYPES[dtype], device="cuda")
    near = T(gen.i8(gen.rng(4), (3, V))).to(x.dtype)
    x[:3] = near
    x[-3:] = near
    t = T(np.array([0, V - 1, 9], np.int64))
    want = iw.speculative.token_logprobs(near, t, top=5, scale=0.1)
    targets = torch.zeros(rows, dtype=torch.int64, device="cuda")
    targets[:3], targets[-3:] = t, t
    got = iw.speculative.token_logprobs(x, targets, top=5, scale=0.1)
    for a, b in zip(got, want):
        for part in (a[:3], a[-3:]):
            if b.dtype == torch.int64:
                assert torch.equal(part, b)
            else:  # few and many blocks share the sums out differently: a few roundings of numbers up to 30
                assert (part - b).abs().max() < 30 * 64 * 2.0 ** -24


def test_empty_batches(iw, gpu):
    sp = iw.speculative
    e = lambda *shape, dtype=torch.int8: torch.empty(shape, dtype=dtype, device="cuda")
    plan = sp.tree_plan(e(0, 8, dtype=torch.int32))
    assert plan.visible.shape == plan.positions.shape == (0, 8)
    q, k, v, ln = e(0, 8, 128), e(0, 2, 32, 64), e(0, 2, 8, 64, 4), e(0, dtype=torch.int32)
    y = sp.tree_attention(q, q, q, k, v, ln, plan.visible, heads=2, qk_multiplier=90, qk_shift=9, frac_bits=8,
                          av_multiplier=100, av_shift=6)
    assert y.shape == (0, 8, 128)
    for lead in ((0,), (0, 3), (3, 0)):
        s = sp.token_logprobs(e(*lead, 100, dtype=torch.float32), e(*lead, dtype=torch.int64), top=2)
        assert s.logprob.shape == s.entropy.shape == lead and s.top_ids.shape == s.top_logprobs.shape == (*lead, 2)


def test_token_logprobs_refuses(iw, gpu):
    f = iw.speculative.token_logprobs
    x = torch.zeros((2, 40), device="cuda")
    for call, what in [(lambda: f(x.double()), "int8, float32"), (lambda: f(x, top=33), "top"), (lambda: f(x, top=-1), "top"),
                       (lambda: f(x[:, :3], top=4), "top"), (lambda: f(x, scale=0.0), "scale"),
                       (lambda: f(x, T(np.zeros(2, np.int32))), "int64"), (lambda: f(x, T(np.zeros(3, np.int64))), "shape"),
                       (lambda: f(x, suppress=T(np.zeros(1, np.int32))), "shape"),
                       (lambda: f(x, suppress=T(np.zeros(2, np.int64))), "int32 or uint32"),
                       (lambda: f(x, torch.zeros(2, dtype=torch.int64)), "GPU")]:
        with pytest.raises(RuntimeError, match=what):
            call()


# ---------------------------------------------------------------------------
# streams, graphs, the whole pass
# ---------------------------------------------------------------------------

def test_captured_round_replays(iw, gpu):
    """Plan, attention, scores and acceptance captured as one graph: every replay on new inputs,
    between eager rounds of the same, gives the eager results."""
    sp = iw.speculative
    B, H, D, cap, N, V = 3, 2, 64, 96, 7, 70000
    c = Case(1, B, H, D, cap, N, [10, 50, 80], [7, 5, 7], "quads")
    C = H * D
    qkv, k, v = T(c.qkv), T(c.k), c.v_view(T(c.vc))
    ln, cnt, par = T(c.lengths), T(c.counts), T(c.parents)
    logits = T(gen.i8(gen.rng(3), (B, N, V)))
    tok = torch.zeros((B, N), dtype=torch.int64, device="cuda")
    caches = sp.TreeCaches([qkv[..., C:2 * C]], [qkv[..., 2 * C:]], [k], [v], heads=H)

    def round_():
        plan = sp.tree_plan(par, cnt, lengths=ln, max_positions=cap)
        y = sp.tree_attention(qkv[..., :C], qkv[..., C:2 * C], qkv[..., 2 * C:], k, v, ln, plan.visible, cnt, heads=H,
                              qk_multiplier=90, qk_shift=9, frac_bits=8, av_multiplier=100, av_shift=6)
        s = sp.token_logprobs(logits, top=3, scale=0.1)
        a = caches.accept(tok, par, s.top_ids[..., 0].contiguous(), ln, cnt)
        return [*plan, y, s.entropy, s.top_ids, s.top_logprobs, *a]

    def eager():
        saved = k.clone(), v.clone()
        out = [t.clone() for t in round_()] + [k.clone(), v.clone()]
        k.copy_(saved[0]), v.copy_(saved[1])
        return out
    eager()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = round_()
    for i in range(4):
        r = gen.rng(100 + i)
        qkv.copy_(T(gen.i8(r, c.qkv.shape)))
        logits.copy_(T(gen.i8(r, (B, N, V))))
        ln.copy_(T(r.integers(0, cap - N, B).astype(np.int32)))
        cnt.copy_(T(r.integers(0, N + 1, B).astype(np.int32)))
        tok.copy_(T(r.integers(0, 3, (B, N))))
        want = eager()
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip([*outs, k, v], want):
            assert torch.equal(a, b) or torch.equal(a.isnan(), b.isnan())


def test_captured_long_cache_replays(iw, gpu):
    """Two graphs of a cache whose keys several blocks share, replayed on two streams at once."""
    B, H, D, cap, N = 2, 2, 128, 2000, 9
    cases = [Case(i, B, H, D, cap, N, [cap, 300 + i], [N, N - 2], "vt") for i in range(2)]
    graphs, got = [], []
    for c in cases:
        c.args = T(c.qkv), T(c.k), T(c.vc), T(c.lengths), T(c.visible), T(c.counts)

    def run(c):
        qkv, k, v, ln, vis, cnt = c.args
        C = H * D
        return iw.speculative.tree_attention(qkv[..., :C], qkv[..., C:2 * C], qkv[..., 2 * C:], k, v, ln, vis, cnt,
                                             heads=H, qk_multiplier=90, qk_shift=9, frac_bits=8, av_multiplier=100,
                                             av_shift=6)
    for c in cases:
        run(c)
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            got.append(run(c))
    streams = [torch.cuda.Stream() for _ in cases]
    for i in range(4):
        for c in cases:
            r = gen.rng(10 * i + cases.index(c))
            c.args[0].copy_(T(gen.i8(r, c.qkv.shape)))
            c.args[3].copy_(T(r.integers(0, cap + 1, B).astype(np.int32)))
        want = [run(c).clone() for c in cases]
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_two_streams_at_once(iw, gpu):
    """Two scores with workspaces of their own, queued on two streams."""
    r = gen.rng(5)
    xs = [T(r.normal(0, 3, (40, 150000)).astype(np.float32)) for _ in range(2)]
    want = [iw.speculative.token_logprobs(x, top=6) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = []
    for _ in range(3):
        for s, x in zip(streams, xs):
            with torch.cuda.stream(s):
                got.append(iw.speculative.token_logprobs(x, top=6))
    torch.cuda.synchronize()
    for i, a in enumerate(got):
        assert all(torch.equal(p, q) for p, q in zip(a[1:], want[i % 2][1:]))


def small_model(iw, heads=6, d=384, vocab=512, text_ctx=48):
    dims = iw.ModelDimensions(n_mels=80, n_audio_ctx=64, n_audio_state=d, n_audio_head=heads, n_audio_layer=2,
                              n_vocab=vocab, n_text_ctx=text_ctx, n_text_state=d, n_text_head=heads, n_text_layer=2)
    P = iw.synth.calibrated_int_params(dims, seed=11)
    return dims, iw.Whisper_int.from_params(dims, P).cuda()


@pytest.mark.parametrize("heads,nodes", [(6, 1), (6, 5), (6, 24), (4, 9)])
def test_tree_decoder_is_greedy_decoding(iw, gpu, heads, nodes):
    """Drafts that are right, wrong and in between: the accepted tokens and the caches are those
    of greedy_decode (heads 4: head_dim 96, V transposed)."""
    print("case: tree decoder", heads, nodes, flush=True)
    dims, model = small_model(iw, heads=heads)
    B, P, steps = 3, 3, 30
    r = gen.rng(nodes)
    mel = iw.synth.synthetic_mel(B, dims.n_mels, 2 * dims.n_audio_ctx, seed=21)
    prompt = T(np.array([[1, 2, 3], [4, 5, 6], [7, 8, 9]], np.int64))
    with torch.no_grad():
        feats = model.embed_audio(T(mel))
        greedy = iw.DecoderRunner(model.decoder, B, dims.n_audio_ctx)
        want = host(iw.greedy_decode(model, feats, prompt, steps, runner=greedy))[:, P:]
        runner = iw.DecoderRunner(model.decoder, B, dims.n_audio_ctx)
        runner.set_audio(feats)
        tree = iw.speculative.TreeDecoder(runner, nodes)
        last = host(tree.start(prompt))
        out = [[int(t)] for t in last]
        rounds = 0
        while min(map(len, out)) < steps:
            rounds += 1
            tokens = r.integers(0, dims.n_vocab, (B, nodes))
            parents = random_tree(r, B, nodes)
            counts = np.array([nodes if len(out[b]) < steps else 0 for b in range(B)], np.int32)
            for b in range(B):
                depth = np.zeros(nodes, int)
                for i in range(1, nodes):
                    depth[i] = depth[parents[b, i]] + 1
                for i in range(nodes):  # most drafts are what greedy decoding gives at that depth
                    at = len(out[b]) - 1 + depth[i]
                    if i == 0 or (at < steps and r.random() < 0.7):
                        tokens[b, i] = want[b, at] if i else out[b][-1]
            res = tree.step(T(tokens), T(parents), T(counts), top=2)
            n, nxt, path = host(res.accept.accepted), host(res.accept.next_token), host(res.accept.path)
            for b in range(B):
                out[b] += [int(tokens[b, j]) for j in path[b, 1:n[b]]] + ([int(nxt[b])] if n[b] else [])
                if n[b]:
                    lg = res.logits[b, path[b, n[b] - 1]].double() * runner.logit_scale
                    assert abs(float(res.scores.top_logprobs[b, path[b, n[b] - 1], 0])
                               - float(lg.log_softmax(0).max())) < 600 * 2.0 ** -24 + 3 * 2.0 ** -24 * 20
        assert [o[:steps] for o in out] == want.tolist()
        if nodes > 1:
            assert rounds < steps - 1
        # what is cached of both: the prompt and the first steps - 1 tokens
        for l in range(dims.n_text_layer):
            n = P + steps - 1
            assert torch.equal(runner.k_self[l][:, :, :n], greedy.k_self[l][:, :, :n])
            a, b = (x.v_self[l].view(tree.v_cache[l].shape) for x in (runner, greedy))
            if runner.v_quads:
                a, b = (x.transpose(3, 4).flatten(2, 3)[:, :, :n] for x in (a, b))
            else:
                a, b = a[..., :n], b[..., :n]
            assert torch.equal(a, b)


def test_tree_decoder_step_replays(iw, gpu):
    """A captured step: its replays on new trees advance the rows as eager steps do."""
    dims, model = small_model(iw)
    B, N, rounds = 2, 5, 6
    mel = iw.synth.synthetic_mel(B, dims.n_mels, 2 * dims.n_audio_ctx, seed=22)
    prompt = T(np.array([[1, 2, 3], [4, 5, 6]], np.int64))
    tokens = torch.zeros((B, N), dtype=torch.int64, device="cuda")
    parents = torch.zeros((B, N), dtype=torch.int32, device="cuda")
    with torch.no_grad():
        feats = model.embed_audio(T(mel))
        runs = []
        for captured in (False, True):
            runner = iw.DecoderRunner(model.decoder, B, dims.n_audio_ctx)
            runner.set_audio(feats)
            tree = iw.speculative.TreeDecoder(runner, N)
            if captured:
                tree.start(prompt)
                tree.step(tokens, parents)
                torch.cuda.synchronize()
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g):
                    res = tree.step(tokens, parents)
            r = gen.rng(9)
            last = tree.start(prompt)
            kept = []
            for _ in range(rounds):
                tokens.copy_(T(r.integers(0, dims.n_vocab, (B, N))))
                tokens[:, 0] = last
                parents.copy_(T(random_tree(r, B, N)))
                if captured:
                    g.replay()
                else:
                    res = tree.step(tokens, parents)
                last = res.accept.next_token.clone()
                kept += [t.clone() for t in (*res.accept, res.logits, tree.lengths)]
                torch.cuda.synchronize()
            assert (tree.lengths >= 3 + rounds).all()
            runs.append(kept)
        assert all(torch.equal(a, b) for a, b in zip(*runs))
