"""The operators of speculative decoding and token scoring: cases, inputs, plain forms.

``listed`` names the cases and ``draw`` makes others of the same ranges;
``prepare`` builds what a program holds before a call, ``run`` is one pass
through an operator (its plain form in elementary torch operations or, where
``own`` is true, the framework's kernels), ``work`` the bytes and operations
that a pass cannot do without and ``exact`` the result restated in 64 bits.

Kinds of cases, the operators of ``i_whisper_amd.speculative``:

* ``attend``  tree_attention: the drafted nodes of every row over its int8 KV cache
              and its own tree
* ``plan``    tree_plan: which node sees which, and the nodes' positions
* ``accept``  TreeCaches.accept: the accepted path, the next token, the path's K/V
              appended to the caches of all layers
* ``score``   token_logprobs: log-probabilities of given tokens, entropy and the
              most probable alternatives of rows of logits

Head counts, widths, vocabulary and contexts are Whisper's five shapes'; the
long cache with wide heads is a generic size.
"""
import math

import torch

own = False

DEVICE = "cuda"
VOCAB = 51865
LOGIT_SCALE = 0.125      # int8 logits times this are the real ones: +-16
ACT = 25.0               # deviation of int8 activations
SHAPES = {"tiny": (4, 4, 96), "base": (6, 8, 64), "small": (12, 12, 64), "medium": (24, 16, 64),
          "large": (32, 20, 64)}  # layers, heads, head_dim
EOT = 50257


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # a short draft for one utterance on the smallest model: latency alone
        _attend("tree_tiny_b1_n5", 1, 4, 96, 448, 40, 80, 5, False),
        # rows of different lengths, one token each: the last step of a batch of drafts
        _attend("tree_medium_b48_n1", 48, 16, 64, 448, 0, 447, 1, True),
        # one utterance with the best model and a bushy draft
        _attend("tree_large_b1_n26", 1, 20, 64, 448, 200, 220, 26, True),
        # the throughput batch, 16 drafted nodes a row
        _attend("tree_large_b128_n16", 128, 20, 64, 448, 16, 432, 16, True),
        # long caches of wide heads, trees that end inside a tile
        _attend("tree_long_b5_n61", 5, 8, 128, 4096, 1000, 4000, 61, False),
        # the plan of one utterance's draft
        _plan("plan_b1_n8", 1, 8),
        # the plan of a full batch's widest trees
        _plan("plan_b128_n64", 128, 64),
        # one utterance's draft accepted into the caches of a small model
        _accept("accept_base_b1_n8", 6, 1, 8, 64, 448, 8, True),
        # a batch's drafts accepted into the caches of twelve layers
        _accept("accept_small_b16_n16", 12, 16, 12, 64, 448, 16, True),
        # one step's alternatives for a beam
        _score("score_b1_int8", 1, VOCAB, "int8", 5, False, False),
        # the words of an utterance scored, as word confidences need them
        _score("score_words_b91_fp32", 91, VOCAB, "float32", 0, True, True),
        # every node of the throughput batch's trees, with its alternatives
        _score("score_tree_b2048_int8", 2048, VOCAB, "int8", 4, True, True),
    ]


def _attend(name, batch, heads, head_dim, cap, lo, hi, nodes, quads):
    return dict(name=name, kind="attend", batch=batch, heads=heads, head_dim=head_dim, cap=cap, lo=lo, hi=hi,
                nodes=nodes, quads=quads)


def _plan(name, batch, nodes):
    return dict(name=name, kind="plan", batch=batch, nodes=nodes)


def _accept(name, layers, batch, heads, head_dim, cap, nodes, quads):
    return dict(name=name, kind="accept", layers=layers, batch=batch, heads=heads, head_dim=head_dim, cap=cap,
                nodes=nodes, quads=quads)


def _score(name, rows, vocab, dtype, top, targets, suppress):
    return dict(name=name, kind="score", rows=rows, vocab=vocab, dtype=dtype, top=top, targets=targets,
                suppress=suppress)


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "score", "score", "plan", "accept"])
    top = max(_cost(c) for c in listed() if c["kind"] == kind)
    while True:
        case = _drawn(kind, rng)
        if _cost(case) <= top:
            return case


def _drawn(kind, rng):
    if kind == "plan":
        case = _plan("", _log(rng, 1, 128), _log(rng, 1, 64))
    elif kind == "score":
        case = _score("", _log(rng, 1, 2048), _log(rng, 1000, 262144),
                      rng.choice(["int8", "float32", "bfloat16", "float16"]), rng.choice([0, 1, 2, 5, 8, 17, 32]),
                      rng.random() < 0.7, rng.random() < 0.5)
    else:
        layers, heads, head_dim = SHAPES[rng.choice(sorted(SHAPES))]
        nodes = _log(rng, 1, 64)
        if kind == "accept":
            case = _accept("", layers, _log(rng, 1, 16), heads, head_dim, 448, nodes, rng.random() < 0.6)
        else:
            cap = 448
            if rng.random() < 0.35:
                heads, head_dim, cap = rng.randint(1, 16), rng.choice([16, 32, 48, 64, 80, 112, 128]), _log(rng, 64, 4096)
            hi = rng.randint(0, cap)
            case = _attend("", _log(rng, 1, 128), heads, head_dim, cap, rng.randint(0, hi), hi, nodes,
                           rng.random() < 0.5)
    del case["name"]
    return case


def _cost(case):
    w = work(case)
    return w["bytes"] / 4e12 + w["flops"] / 5e14


def work(case):
    b, n = case.get("batch"), case.get("nodes")
    if case["kind"] == "plan":
        return {"bytes": b * (n * (4 + 8 + 4) + 8), "flops": b * n * 8}
    if case["kind"] == "score":
        r, v, k = case["rows"], case["vocab"], case["top"]
        item = torch.empty(0, dtype=getattr(torch, case["dtype"])).element_size()
        return {"bytes": r * (v * item + 8 * case["targets"] + 8 + 12 * k) + v // 8 * case["suppress"], "flops": r * v * 6}
    c = case["heads"] * case["head_dim"]
    if case["kind"] == "accept":
        # about two nodes of a draft are accepted: K and V read once and written once
        return {"bytes": b * (n * 24 + 28) + case["layers"] * b * 2 * c * 4, "flops": b * n * 8}
    keys = (case["lo"] + case["hi"]) / 2  # cached keys of an average row
    return {"bytes": int(b * (2 * c * keys + 4 * n * c + 8 * n + 4)), "flops": int(4 * b * n * c * (keys + (n + 1) / 4))}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _act(g, *shape):
    return (torch.randn(shape, generator=g, device=DEVICE) * ACT).round_().clamp_(-127, 127).to(torch.int8)


def _tree(g, batch, nodes):
    """Parents of random trees: node 0 is the root, node i hangs on an earlier node, mostly a near one."""
    back = (torch.rand((batch, nodes), generator=g, device=DEVICE).pow(2.0)
            * torch.arange(nodes, device=DEVICE)).long() + 1
    parent = torch.arange(nodes, device=DEVICE) - back
    parent[:, 0] = -1
    return parent.clamp_(min=0).where(torch.arange(nodes, device=DEVICE) > 0, -torch.ones_like(parent)).to(torch.int32)


def _counts(g, batch, nodes):
    """Nodes in use: some rows have shorter drafts."""
    short = torch.randint(1, nodes + 1, (batch,), generator=g, device=DEVICE)
    cut = torch.rand(batch, generator=g, device=DEVICE) < 0.3
    return torch.where(cut, short, torch.full_like(short, nodes)).to(torch.int32)


def _closure(parents, counts):
    """visible[b, i, j]: node j is node i or one of its ancestors, both in use."""
    b, n = parents.shape
    seen = torch.zeros((b, n, n), dtype=torch.bool, device=DEVICE)
    rows = torch.arange(b, device=DEVICE)
    for i in range(n):
        p = parents[:, i].long()
        seen[:, i] = torch.where((p >= 0)[:, None], seen[rows, p.clamp(min=0)], False)
        seen[:, i, i] = True
    used = torch.arange(n, device=DEVICE) < counts[:, None]
    return seen & used[:, :, None] & used[:, None, :]


def _inputs(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    if case["kind"] == "score":
        return _score_inputs(case, g)
    b, n = case["batch"], case["nodes"]
    s = {"parents": _tree(g, b, n), "counts": _counts(g, b, n)}
    if case["kind"] == "plan":
        s["lengths"] = torch.randint(0, 448, (b,), generator=g, device=DEVICE, dtype=torch.int32)
        s["max_positions"] = 448
        return s
    h, d, cap = case["heads"], case["head_dim"], case["cap"]
    c, tp = h * d, (cap + 15) // 16 * 16

    def caches():
        v = (b, h, tp // 4, d, 4) if case["quads"] else (b, h, d, tp)
        return _act(g, b, h, cap, d), _act(g, *v)

    if case["kind"] == "attend":
        qkv = _act(g, b, n, 3 * c)  # the fused projection's rows
        s["q"], s["k_new"], s["v_new"] = qkv[..., :c], qkv[..., c:2 * c], qkv[..., 2 * c:]
        s["k_cache"], s["v_cache"] = caches()
        s["lengths"] = torch.randint(case["lo"], case["hi"] + 1, (b,), generator=g, device=DEVICE, dtype=torch.int32)
        bits = torch.ones((), dtype=torch.int64, device=DEVICE) << torch.arange(n, device=DEVICE)
        s["visible"] = (_closure(s["parents"], s["counts"]) * bits).sum(-1)
        # scores of deviation 2 in the real scale, as a calibrated layer requantises them
        frac = 8
        m = 2.0 * 2 ** frac / (math.sqrt(d) * ACT * ACT)
        shift = 0
        while m < 64:
            m, shift = 2 * m, shift + 1
        s["scalars"] = dict(qk_multiplier=round(m), qk_shift=shift, frac_bits=frac, av_multiplier=128, av_shift=6,
                            rsqrt_offset=16)
        return s
    layers = [(_act(g, b, n, 3 * c), caches()) for _ in range(case["layers"])]
    s["k_new"] = [q[..., c:2 * c] for q, _ in layers]
    s["v_new"] = [q[..., 2 * c:] for q, _ in layers]
    s["k_cache"] = [kv[0] for _, kv in layers]
    s["v_cache"] = [kv[1] for _, kv in layers]
    s["lengths"] = torch.randint(0, cap - n + 1, (b,), generator=g, device=DEVICE, dtype=torch.int32)
    s["tokens"] = torch.randint(0, VOCAB, (b, n), generator=g, device=DEVICE)
    # the model's choice after a node: often the token of a node that hangs on it
    s["choice"] = torch.randint(0, VOCAB, (b, n), generator=g, device=DEVICE)
    agrees = torch.rand((b, n), generator=g, device=DEVICE) < 0.6
    rows = torch.arange(b, device=DEVICE)
    for j in range(1, n):
        p = s["parents"][:, j].long()
        s["choice"][rows, p] = torch.where(agrees[:, j], s["tokens"][:, j], s["choice"][rows, p])
    s["choice"][torch.rand((b, n), generator=g, device=DEVICE) < 0.02] = EOT
    return s


def _score_inputs(case, g):
    r, v = case["rows"], case["vocab"]
    x = torch.randn((r, v), generator=g, device=DEVICE) * 2.0 - 4.0
    # a few candidates a row stand out, by far or by little
    cand = torch.randint(0, v, (r, 6), generator=g, device=DEVICE)
    x.scatter_add_(1, cand, 4.0 + 14.0 * torch.rand((r, 6), generator=g, device=DEVICE))
    s = {"scale": 1.0, "top": case["top"], "targets": None, "suppress": None}
    if case["dtype"] == "int8":
        s["scale"] = LOGIT_SCALE
        s["logits"] = (x / LOGIT_SCALE).round_().clamp_(-127, 127).to(torch.int8)
    else:
        s["logits"] = x.to(getattr(torch, case["dtype"]))
    if case["targets"]:
        other = torch.randint(0, v, (r,), generator=g, device=DEVICE)
        s["targets"] = torch.where(torch.rand(r, generator=g, device=DEVICE) < 0.75, cand[:, 0], other)
    if case["suppress"]:
        # the decoding task's suppressed tokens, as the words of a bit mask
        off = torch.zeros((v + 31) // 32 * 32, dtype=torch.int64, device=DEVICE)
        off[torch.randint(0, v, (90,), generator=g, device=DEVICE)] = 1
        words = (off.view(-1, 32) << torch.arange(32, device=DEVICE)).sum(-1)
        s["suppress"] = torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)
        if s["targets"] is not None:  # targets are tokens that may be chosen
            s["targets"] = torch.where(off[s["targets"]] == 0, s["targets"], off[:v].argmin())
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        import __graft_entry__
        s["ops"] = __graft_entry__.load_package().speculative
        if case["kind"] == "accept":
            s["caches"] = s["ops"].TreeCaches(s["k_new"], s["v_new"], s["k_cache"], s["v_cache"], heads=case["heads"])
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(s):
    kind = s["case"]["kind"]
    if not own:
        return {"plan": _plain_plan, "attend": _plain_attend, "accept": _plain_accept, "score": _plain_score}[kind](s)
    ops = s["ops"]
    if kind == "plan":
        return list(ops.tree_plan(s["parents"], s["counts"], lengths=s["lengths"], max_positions=s["max_positions"]))
    if kind == "attend":
        return ops.tree_attention(s["q"], s["k_new"], s["v_new"], s["k_cache"], s["v_cache"], s["lengths"],
                                  s["visible"], s["counts"], heads=s["case"]["heads"], **s["scalars"])
    if kind == "accept":
        a = s["caches"].accept(s["tokens"], s["parents"], s["choice"], s["lengths"], s["counts"], eot=EOT)
        return [a.path, a.accepted, a.next_token, a.lengths, *s["k_cache"], *s["v_cache"]]
    t = ops.token_logprobs(s["logits"], s["targets"], top=s["top"], scale=s["scale"], suppress=s["suppress"])
    return [x for x in (t.logprob, t.entropy, t.top_ids, t.top_logprobs) if x is not None]


def _plain_plan(s):
    parents, counts = s["parents"].long(), s["counts"]
    b, n = parents.shape
    rows = torch.arange(b, device=parents.device)
    used = torch.arange(n, device=parents.device) < counts[:, None]
    visible = torch.zeros((b, n), dtype=torch.int64, device=parents.device)
    depth = torch.zeros((b, n), dtype=torch.int64, device=parents.device)
    for i in range(n):
        p = parents[:, i]
        has, at = p >= 0, p.clamp(min=0)
        visible[:, i] = torch.where(has, visible[rows, at], 0) | (1 << i if i < 63 else -2 ** 63)
        depth[:, i] = torch.where(has, depth[rows, at] + 1, 0)
    visible = torch.where(used, visible, 0)
    pos = (s["lengths"][:, None] + torch.where(used, depth, 0)).clamp(max=s["max_positions"] - 1)
    return [visible, pos.to(torch.int32)]


def _rshift(x, n):
    """x / 2^n, halves away from zero, modulo 2^32."""
    if n == 0:
        return x
    return _wrap(x + (1 << (n - 1)) - (x < 0).long()) >> n


def _wrap(x):
    return ((x + 2 ** 31) & 0xFFFFFFFF) - 2 ** 31


def _inv_sqrt(x, off):
    """The integer inverse square root: the bits of float32(x) give the first guess, two Newton steps."""
    e = torch.zeros_like(x)
    for step in (16, 8, 4, 2, 1):
        more = (x >> (e + step)) > 0
        e = torch.where(more, e + step, e)
    sig = torch.where(e <= 23, x << (23 - e).clamp(min=0), x >> (e - 23).clamp(min=0))
    i = torch.where(x == 0, 0, ((e + 127) << 23) | (sig & 0x7FFFFF))
    raw = (0x5F3759DF - (i >> 1) + (off << 23)) & 0xFFFFFFFF
    e = ((raw >> 23) & 0xFF) - 127
    sig = (1 << 23) | (raw & 0x7FFFFF)
    y = torch.where(e >= 23, sig << (e - 23).clamp(min=0), sig >> (23 - e).clamp(0, 62))
    y = _wrap(torch.where(e < 0, 0, y))
    for _ in range(2):
        t = _wrap(_rshift(_wrap(x * y), off) * y)
        y = _rshift(_wrap(y * _wrap((3 << off) - t)), off + 1)
    return y


def _shift_exp(n, f):
    """The shift exponential of -n, n in [0, 65535], in 16-bit arithmetic."""
    def w16(v):
        return ((v + 2 ** 15) & 0xFFFF) - 2 ** 15
    x = w16(-n)
    fix = w16(w16(x + (x >> 1)) - (x >> 4))
    whole = fix >> f
    num = (1 << f) + ((fix - (whole << f)) >> 1)
    e = torch.where((whole > 0) | (whole <= -16), 0, num >> (-whole).clamp(0, 15))
    return torch.where(x > 0, 0, e >> max(f - 7, 0))


def _plain_attend(s):
    case, sc = s["case"], s["scalars"]
    b, n, h, d, cap = case["batch"], case["nodes"], case["heads"], case["head_dim"], case["cap"]
    dev = s["q"].device

    def heads(x):
        return x.reshape(b, n, h, d).transpose(1, 2)
    v = s["v_cache"]
    v = v.transpose(3, 4).reshape(b, h, -1, d) if v.dim() == 5 else v.transpose(2, 3)
    k = torch.cat([s["k_cache"], heads(s["k_new"])], 2).float().view(b * h, cap + n, d)
    v = torch.cat([v[:, :, :cap], heads(s["v_new"])], 2).double().view(b * h, cap + n, d)
    q = heads(s["q"]).float().reshape(b * h, n, d)
    used = torch.arange(n, device=dev) < s["counts"][:, None]
    bits = (s["visible"][:, :, None] >> torch.arange(n, device=dev)) & 1 > 0
    sees = torch.cat([(torch.arange(cap, device=dev) < s["lengths"][:, None])[:, None].expand(b, n, cap),
                      bits & used[:, None]], 2) & used[:, :, None]
    sees = sees[:, None]  # of every head
    # products of up to 128 terms below 2^14 are exact in 32 bits
    score = torch.bmm(q, k.transpose(1, 2).contiguous()).long().view(b, h, n, cap + n)
    score = _rshift(_wrap(score * sc["qk_multiplier"]), sc["qk_shift"]).clamp(-32768, 32767)
    top = torch.where(sees, score, -32768).amax(-1, keepdim=True)
    p = torch.where(sees, _shift_exp((top + 1 - score) & 0xFFFF, sc["frac_bits"]), 0)
    total = p.sum(-1, keepdim=True)
    o = torch.bmm(p.double().view(b * h, n, cap + n), v).long().view(b, h, n, d)  # sums pass 2^24
    inv, off = _inv_sqrt(total, sc["rsqrt_offset"]), sc["rsqrt_offset"]
    y = _rshift(_wrap(_rshift(_wrap(_wrap(o) * inv), off) * inv), off)
    y = _rshift(_wrap(y * sc["av_multiplier"]), sc["av_shift"]).clamp(-127, 127).to(torch.int8)
    return y.transpose(1, 2).reshape(b, n, h * d)


def _plain_accept(s):
    case = s["case"]
    b, n, cap = case["batch"], case["nodes"], case["cap"]
    dev = s["tokens"].device
    rows = torch.arange(b, device=dev)
    lengths, counts = s["lengths"].long(), s["counts"].long()
    room = cap - lengths
    path = torch.full((b, n), -1, dtype=torch.int64, device=dev)
    taken = ((counts > 0) & (room > 0)).long()
    path[:, 0] = torch.where(taken > 0, 0, -1)
    cur = torch.zeros_like(lengths)
    for j in range(1, n):
        want = s["choice"][rows, cur]
        hit = ((s["parents"][:, j] == cur) & (s["tokens"][:, j] == want) & (want != EOT) & (j < counts)
               & (taken > 0) & (taken < room))
        at = taken.clamp(max=n - 1)
        path[rows, at] = torch.where(hit, j, path[rows, at])
        taken = taken + hit
        cur = torch.where(hit, j, cur)
    after = torch.where(taken > 0, s["choice"][rows, cur], -1)
    row, col = (path >= 0).nonzero(as_tuple=True)
    node, slot = path[row, col], lengths[row] + col
    h, d = case["heads"], case["head_dim"]
    for kn, vn, kc, vc in zip(s["k_new"], s["v_new"], s["k_cache"], s["v_cache"]):
        kc[row, :, slot] = kn[row, node].view(-1, h, d)
        if vc.dim() == 5:
            vc[row, :, slot // 4, :, slot % 4] = vn[row, node].view(-1, h, d)
        else:
            vc[row, :, :, slot] = vn[row, node].view(-1, h, d)
    return [path.to(torch.int32), taken.to(torch.int32), after, (lengths + taken).to(torch.int32), *s["k_cache"],
            *s["v_cache"]]


def _plain_score(s):
    raw, top = s["logits"].float(), s["top"]
    v = raw.shape[1]
    if s["suppress"] is not None:
        i = torch.arange(v, device=raw.device)
        raw = raw.masked_fill((s["suppress"][i >> 5] >> (i & 31)) & 1 > 0, -math.inf)
    x = raw * s["scale"]
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    # the sums of a whole vocabulary, and what is small next to its largest term, in 64 bits
    z = e.double().sum(-1)
    lse = torch.log(z)
    spread = torch.where(e > 0, e * (m - x), 0).double().sum(-1)
    out = []
    if s["targets"] is not None:
        at = x.gather(1, s["targets"][:, None])[:, 0]
        out.append(((at - m[:, 0]).double() - lse).float())
    out.append((lse + spread / z).float())
    if top:
        # the order of values as that of whole numbers, ties to the lowest index
        bits = (raw + 0.0).view(torch.int32).long()
        key = torch.where(bits >= 0, bits, -(bits & 0x7FFFFFFF)) << 32
        ids = (key + (v - 1 - torch.arange(v, device=raw.device))).topk(top, -1).indices
        out += [ids, ((x.gather(1, ids) - m).double() - lse[:, None]).float()]
    return out


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = _inputs(case, seed)
    return {"plan": _exact_plan, "attend": _exact_attend, "accept": _exact_accept, "score": _exact_score}[case["kind"]](case, s)


def _exact_plan(case, s):
    # paths walked node by node on the host
    parents, counts, lengths = s["parents"].tolist(), s["counts"].tolist(), s["lengths"].tolist()
    visible, pos = [], []
    for par, cnt, ln in zip(parents, counts, lengths):
        vis, at = [0] * len(par), [min(ln, 447)] * len(par)
        for i in range(cnt):
            j, deep = i, -1
            while j >= 0:
                vis[i] |= 1 << j
                j, deep = par[j], deep + 1
            vis[i] -= (vis[i] >> 63) << 64
            at[i] = min(ln + deep, 447)
        visible.append(vis)
        pos.append(at)
    return [torch.tensor(visible, dtype=torch.int64), torch.tensor(pos, dtype=torch.int32)]


def _exact_attend(case, s):
    # row by row, over the keys that the row has, its probabilities from a table of all 65536 differences
    b, n, h, d = case["batch"], case["nodes"], case["heads"], case["head_dim"]
    sc = s["scalars"]
    f = sc["frac_bits"]
    table = []
    for diff in range(65536):
        x = -diff if diff <= 32768 else 65536 - diff
        fix = x + x // 2 - x // 16
        if x > 0 or fix < -32768:  # 16 bits wrap: these are far below the maximum
            table.append(0)
            continue
        whole = fix // 2 ** f
        table.append(0 if -whole >= 16 else ((2 ** f + (fix - whole * 2 ** f) // 2) >> -whole) >> max(f - 7, 0))
    table = torch.tensor(table, dtype=torch.float64, device=DEVICE)

    def shr(x, bits):
        half = 2 ** bits // 2
        return torch.where(x < 0, -((-x + half) >> bits), (x + half) >> bits)
    out = torch.zeros((b, n, h * d), dtype=torch.int8, device=DEVICE)
    for i in range(b):
        cnt, ln = int(s["counts"][i]), int(s["lengths"][i])
        v = s["v_cache"][i]
        v = v.permute(0, 1, 3, 2).reshape(h, -1, d) if v.dim() == 4 else v.transpose(1, 2)
        q, k, w = (s[x][i, :cnt].view(cnt, h, d).transpose(0, 1).double() for x in ("q", "k_new", "v_new"))
        k = torch.cat([s["k_cache"][i, :, :ln].double(), k], 1)
        w = torch.cat([v[:, :ln].double(), w], 1)
        sees = torch.ones((cnt, ln + cnt), dtype=torch.bool, device=DEVICE)
        for j in range(cnt):
            sees[:, ln + j] = (s["visible"][i, :cnt] >> j) % 2 == 1
        score = shr((q @ k.transpose(1, 2).contiguous()).long() * sc["qk_multiplier"], sc["qk_shift"]).clamp(-32768, 32767)
        best = score.masked_fill(~sees, -32768).amax(-1, keepdim=True)
        p = table[(best + 1 - score) % 65536] * sees
        o, total = (p @ w).long(), p.sum(-1, keepdim=True).long()
        inv = _inv_sqrt_host(total, sc["rsqrt_offset"])
        y = shr(_wrap(o * inv), sc["rsqrt_offset"])
        y = shr(_wrap(y * inv), sc["rsqrt_offset"])
        y = shr(_wrap(y * sc["av_multiplier"]), sc["av_shift"]).clamp(-127, 127)
        out[i, :cnt] = y.transpose(0, 1).reshape(cnt, h * d).to(torch.int8)
    return out


def _inv_sqrt_host(total, off):
    """The integer inverse square root of whole numbers, one at a time."""
    import struct

    def w32(v):
        return (v + 2 ** 31) % 2 ** 32 - 2 ** 31

    def shr(v, bits):
        return w32(v + 2 ** bits // 2 - (v < 0)) >> bits

    def one(x):
        # float32(x) cut off below its 24th bit
        cut = x if x < 2 ** 24 else x >> (x.bit_length() - 24) << (x.bit_length() - 24)
        i = struct.unpack("<i", struct.pack("<f", float(cut)))[0]
        raw = (0x5F3759DF - (i >> 1) + (off << 23)) % 2 ** 32
        e = ((raw >> 23) & 0xFF) - 127
        y = 0 if e < 0 else w32((2 ** 23 + raw % 2 ** 23) * 2 ** e >> 23)
        for _ in range(2):
            t = w32(shr(w32(x * y), off) * y)
            y = shr(w32(y * w32(3 * 2 ** off - t)), off + 1)
        return y
    values, back = total.unique(return_inverse=True)
    return torch.tensor([one(x) for x in values.tolist()], dtype=torch.int64, device=total.device)[back]


def _exact_accept(case, s):
    b, n, cap, h, d = (case[x] for x in ("batch", "nodes", "cap", "heads", "head_dim"))
    tokens, parents, choice, counts, lengths = (s[x].tolist() for x in ("tokens", "parents", "choice", "counts", "lengths"))
    paths, after = [], []
    for i in range(b):
        path = [0] if counts[i] > 0 and lengths[i] < cap else []
        while path and choice[i][path[-1]] != EOT and lengths[i] + len(path) < cap:
            nxt = [j for j in range(path[-1] + 1, counts[i])
                   if parents[i][j] == path[-1] and tokens[i][j] == choice[i][path[-1]]]
            if not nxt:
                break
            path.append(nxt[0])
        after.append(choice[i][path[-1]] if path else -1)
        paths.append(path)
    for layer in range(case["layers"]):
        for i, path in enumerate(paths):
            ln = lengths[i]
            idx = torch.tensor(path, dtype=torch.int64, device=DEVICE)
            s["k_cache"][layer][i, :, ln:ln + len(path)] = s["k_new"][layer][i, idx].view(-1, h, d).transpose(0, 1)
            v = s["v_new"][layer][i, idx].view(-1, h, d).permute(1, 2, 0)
            if case["quads"]:
                flat = s["v_cache"][layer][i].transpose(1, 2).reshape(h, d, -1)
                flat[:, :, ln:ln + len(path)] = v
                s["v_cache"][layer][i] = flat.view(h, d, -1, 4).transpose(1, 2)
            else:
                s["v_cache"][layer][i, :, :, ln:ln + len(path)] = v
    return [torch.tensor([p + [-1] * (n - len(p)) for p in paths], dtype=torch.int32),
            torch.tensor([len(p) for p in paths], dtype=torch.int32), torch.tensor(after, dtype=torch.int64),
            torch.tensor([ln + len(p) for ln, p in zip(lengths, paths)], dtype=torch.int32), *s["k_cache"], *s["v_cache"]]


def _exact_score(case, s):
    x = s["logits"].double()
    if s["suppress"] is not None:
        bits = [(w >> j) & 1 for w in s["suppress"].tolist() for j in range(32)][:case["vocab"]]
        x[:, torch.tensor(bits, device=DEVICE) == 1] = -math.inf
    x *= s["scale"]
    order = x.sort(dim=-1, descending=True, stable=True)
    best = order.values[:, :1]
    rest = torch.exp(order.values[:, 1:] - best)
    z = rest.sum(-1, keepdim=True)  # next to the largest term's 1
    low = torch.where(rest > 0, rest * (best - order.values[:, 1:]), 0).sum(-1, keepdim=True)
    lse = torch.log1p(z)
    out = []
    if s["targets"] is not None:
        out.append((x.gather(1, s["targets"][:, None]) - best - lse)[:, 0])
    out.append((lse + low / (1 + z))[:, 0])
    if s["top"]:
        out += [order.indices[:, :s["top"]], order.values[:, :s["top"]] - best - lse]
    return out
