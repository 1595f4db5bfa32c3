"""The operators of sampled decoding with the model's own drafts: cases, inputs, plain forms.

``listed`` names the cases and ``draw`` makes others of the same ranges;
``prepare`` builds what a program holds before a call, ``run`` is one pass
through an operator (its plain form in elementary torch operations or, where
``own`` is true, the framework's kernels), ``work`` the bytes and operations
that a pass cannot do without and ``exact`` the result restated in 64 bits.

Kinds of cases, the operators of ``i_whisper_amd.drafts``:

* ``window``  window_attention: integer attention of each query over the keys around
              its position and a few first ones, over int8 caches or projected rows
* ``sample``  sample_tokens: a token of each row of logits, drawn by a given random number
* ``verify``  verify_drafts: the drafted tokens of each row accepted or replaced against the
              model's probabilities, by given random numbers

Head counts, widths, vocabulary and contexts are Whisper's five shapes'; the
long caches with wide heads are generic sizes.
"""
import math

import torch

own = False

DEVICE = "cuda"
VOCAB = 51865
LOGIT_SCALE = 0.125      # int8 logits times this are the real ones: +-16
ACT = 25.0               # deviation of int8 activations
SHAPES = {"tiny": (4, 96), "base": (8, 64), "small": (12, 64), "medium": (16, 64), "large": (20, 64)}  # heads, head_dim
TEMPERATURES = (0.0, 0.2, 0.4, 0.6, 0.8, 1.0)  # the decoding task's fallback


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # a drafted token of one utterance on the smallest model: latency alone
        _window("window_tiny_b1_n1", 1, 4, 96, 448, 100, 440, 1, 63, 0, 4, "vt", False),
        # a drafted token of the throughput batch, rows of different lengths
        _window("window_large_b128_n1", 128, 20, 64, 448, 8, 447, 1, 127, 0, 4, "quads", False),
        # the same step's cross-attention: the audio frames around where each row is
        _window("window_cross_large_b128", 128, 20, 64, 1500, 1500, 1500, 1, 128, 128, 8, "vt", True),
        # the encoder of one utterance with local attention, for low latency
        _window("window_encoder_base_b1", 1, 8, 64, 1500, 1500, 1500, 1500, 127, 127, 0, "rows", False),
        # a batch through the largest encoder with local attention
        _window("window_encoder_large_b16", 16, 20, 64, 1500, 1500, 1500, 1500, 255, 255, 16, "rows", False),
        # a long text's prompt, causal, wide heads
        _window("window_prompt_b2_n8192", 2, 8, 128, 8192, 8192, 8192, 8192, 1023, 0, 4, "vt", False),
        # one token of a few rows over very long caches
        _window("window_long_b4_n1", 4, 8, 128, 65536, 30000, 65000, 1, 4095, 0, 64, "quads", False),
        # a token of one utterance
        _sample("sample_b1_int8", 1, VOCAB, "int8", False, False),
        # a token after every node of the throughput batch's trees, each row at its own temperature
        _sample("sample_tree_b2048_bf16", 2048, VOCAB, "bfloat16", True, True),
        # four drafted tokens of one utterance
        _verify("verify_b1_n5_int8", 1, 5, VOCAB, "int8", True, False, False),
        # drafts of a batch of float models, rows at different temperatures, suppressed tokens
        _verify("verify_b24_n6_fp32", 24, 6, VOCAB, "float32", True, True, True),
        # the throughput batch's drafts
        _verify("verify_b128_n8_int8", 128, 8, VOCAB, "int8", True, False, True),
    ]


def _window(name, batch, heads, head_dim, cap, lo, hi, queries, before, after, sinks, layout, frames):
    """``layout``: V transposed ("vt") or in key quads ("quads") beside K per head, or K as rows of a fused
    projection and V transposed ("rows"); ``frames``: the queries' positions are given."""
    return dict(name=name, kind="window", batch=batch, heads=heads, head_dim=head_dim, cap=cap, lo=lo, hi=hi,
                queries=queries, before=before, after=after, sinks=sinks, layout=layout, frames=frames)


def _sample(name, rows, vocab, dtype, mixed, suppress):
    """``mixed``: every row has a temperature of its own."""
    return dict(name=name, kind="sample", rows=rows, vocab=vocab, dtype=dtype, mixed=mixed, suppress=suppress)


def _verify(name, batch, nodes, vocab, dtype, drawn, mixed, suppress):
    """``drawn``: the drafts were drawn from a model's logits, else they are given tokens (of an earlier window)."""
    return dict(name=name, kind="verify", batch=batch, nodes=nodes, vocab=vocab, dtype=dtype, drawn=drawn,
                mixed=mixed, suppress=suppress)


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng):
    kind = rng.choice(["window", "window", "sample", "verify"])
    top = max(_cost(c) for c in listed() if c["kind"] == kind)
    while True:
        case = _drawn(kind, rng)
        if _cost(case) <= top:
            return case


def _drawn(kind, rng):
    if kind == "sample":
        case = _sample("", _log(rng, 1, 2048), _log(rng, 1000, 262144),
                       rng.choice(["int8", "float32", "bfloat16", "float16"]), rng.random() < 0.5, rng.random() < 0.5)
    elif kind == "verify":
        case = _verify("", _log(rng, 1, 128), _log(rng, 1, 16), _log(rng, 1000, 262144),
                       rng.choice(["int8", "float32", "bfloat16", "float16"]), rng.random() < 0.75, rng.random() < 0.5,
                       rng.random() < 0.5)
    else:
        heads, head_dim = SHAPES[rng.choice(sorted(SHAPES))]
        if rng.random() < 0.4:
            heads, head_dim = rng.randint(1, 16), rng.choice([16, 32, 48, 64, 80, 112, 128])
        how = rng.choice(["token", "token", "frames", "prompt", "encoder"])
        batch = _log(rng, 1, 128)
        before, after, sinks, queries, layout = _log(rng, 1, 2048) - 1, 0, rng.choice([0, 1, 4, 16, 70]), 1, "vt"
        if how == "encoder":
            cap = queries = _log(rng, 64, 3000)
            lo = hi = cap
            after, layout = rng.choice([before, 0, before // 3]), "rows"
        elif how == "prompt":
            cap = _log(rng, 16, 8192)
            hi = rng.randint(1, cap)
            lo, queries = rng.randint(max(1, hi // 2), hi), _log(rng, 2, hi + 1)
            layout = rng.choice(["vt", "quads"])
        else:
            cap = _log(rng, 64, 65536)
            hi = rng.randint(1, cap)
            lo, queries = rng.randint(0, hi), rng.choice([1, 1, 1, 4, 8])
            layout = rng.choice(["vt", "quads"])
            after = before if how == "frames" else 0
        if batch * heads * cap * head_dim > 1 << 31:
            batch = max(1, (1 << 31) // (heads * cap * head_dim))
        case = _window("", batch, heads, head_dim, cap, lo, hi, queries, before, after, sinks, layout,
                       how == "frames")
    del case["name"]
    return case


def _cost(case):
    w = work(case)
    return w["bytes"] / 4e12 + w["flops"] / 2e14


def _seen(case):
    """Of a row of average length: visible (query, key) pairs and the keys that any query sees."""
    length, n = (case["lo"] + case["hi"]) // 2, case["queries"]
    pairs, first, last = 0, length, 0
    for i in range(n):
        p = length // 2 if case["frames"] else length - n + i
        end = min(length, p + case["after"] + 1)
        start = max(0, min(p - case["before"], end))
        if end > start:
            first, last = min(first, start), max(last, end)
        pairs += max(0, end - start) + max(0, min(case["sinks"], start, end))
    return pairs, max(0, last - first) + max(0, min(case["sinks"], first))


def work(case):
    if case["kind"] == "window":
        b, n, h, d = case["batch"], case["queries"], case["heads"], case["head_dim"]
        pairs, keys = _seen(case)
        return {"bytes": b * h * (2 * d * keys + 2 * d * n) + 4 * b, "flops": 4 * b * h * d * pairs}
    item = torch.empty(0, dtype=getattr(torch, case["dtype"])).element_size()
    v = case["vocab"]
    if case["kind"] == "sample":
        r = case["rows"]
        return {"bytes": r * (v * item + 16 + 4 * case["mixed"]), "flops": r * v * 8}
    b, n = case["batch"], case["nodes"]
    rows = b * (n + (n - 1) * case["drawn"])
    return {"bytes": rows * v * item + b * (n * 20 + 20), "flops": rows * v * 8}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _act(g, *shape):
    return (torch.randn(shape, generator=g, device=DEVICE) * ACT).round_().clamp_(-127, 127).to(torch.int8)


def _inputs(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    return {"window": _window_inputs, "sample": _sample_inputs, "verify": _verify_inputs}[case["kind"]](case, g)


def _window_inputs(case, g):
    b, n, h, d, cap = (case[x] for x in ("batch", "queries", "heads", "head_dim", "cap"))
    c, tp = h * d, (cap + 15) // 16 * 16
    s = {}
    qkv = _act(g, b, n, 3 * c)  # the fused projection's rows
    s["q"] = qkv[..., :c]
    if case["layout"] == "rows":
        s["k"] = qkv[..., c:2 * c].unflatten(2, (h, d)).transpose(1, 2)
    else:
        s["k"] = _act(g, b, h, cap, d)
    s["v"] = _act(g, b, h, tp // 4, d, 4) if case["layout"] == "quads" else _act(g, b, h, d, tp)
    s["lengths"] = s["positions"] = None
    if case["layout"] != "rows":
        s["lengths"] = torch.randint(case["lo"], case["hi"] + 1, (b,), generator=g, device=DEVICE, dtype=torch.int32)
    if case["frames"]:  # where each row is, its queries a few frames apart
        at = torch.rand((b, 1), generator=g, device=DEVICE) * s["lengths"][:, None]
        s["positions"] = (at.long() + 3 * torch.arange(n, device=DEVICE)).to(torch.int32)
    # scores of deviation 2 in the real scale, as a calibrated layer requantises them
    frac = 8
    m = 2.0 * 2 ** frac / (math.sqrt(d) * ACT * ACT)
    shift = 0
    while m < 64:
        m, shift = 2 * m, shift + 1
    s["scalars"] = dict(qk_multiplier=round(m), qk_shift=shift, frac_bits=frac, av_multiplier=128, av_shift=6,
                        rsqrt_offset=16)
    return s


def _logits(g, rows, v):
    """Real logits of rows: a few candidates stand out, by far or by little."""
    x = torch.randn((rows, v), generator=g, device=DEVICE) * 2.0 - 4.0
    cand = torch.randint(0, v, (rows, 6), generator=g, device=DEVICE)
    return x.scatter_add_(1, cand, 4.0 + 14.0 * torch.rand((rows, 6), generator=g, device=DEVICE))


def _held(x, dtype):
    """Real logits as a model leaves them."""
    if dtype == "int8":
        return (x / LOGIT_SCALE).round_().clamp_(-127, 127).to(torch.int8)
    return x.to(getattr(torch, dtype))


def _suppressed(g, v):
    """The decoding task's suppressed tokens, as the words of a bit mask and as truth values."""
    off = torch.zeros((v + 31) // 32 * 32, dtype=torch.int64, device=DEVICE)
    off[torch.randint(0, v, (90,), generator=g, device=DEVICE)] = 1
    words = (off.view(-1, 32) << torch.arange(32, device=DEVICE)).sum(-1)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32), off[:v] > 0


def _temperature(case, g, rows):
    if not case["mixed"]:
        return 0.8
    pick = torch.randint(0, len(TEMPERATURES), (rows,), generator=g, device=DEVICE)
    return torch.tensor(TEMPERATURES, device=DEVICE)[pick]


def _sample_inputs(case, g):
    r, v = case["rows"], case["vocab"]
    s = {"scale": LOGIT_SCALE if case["dtype"] == "int8" else 1.0, "suppress": None}
    s["logits"] = _held(_logits(g, r, v), case["dtype"])
    s["uniforms"] = torch.rand(r, generator=g, device=DEVICE)
    s["temperature"] = _temperature(case, g, r)
    if case["suppress"]:
        s["suppress"] = _suppressed(g, v)[0]
    return s


def _verify_inputs(case, g):
    b, n, v = case["batch"], case["nodes"], case["vocab"]
    s = {"scale": LOGIT_SCALE if case["dtype"] == "int8" else 1.0, "suppress": None, "draft_logits": None}
    s["temperature"] = t = _temperature(case, g, b)
    off = None
    if case["suppress"]:
        s["suppress"], off = _suppressed(g, v)
    x = _logits(g, b * n, v).view(b, n, v)
    # a weaker model of the same text: its logits are off by about one
    draft = _held(x[:, :n - 1] + torch.randn((b, n - 1, v), generator=g, device=DEVICE), case["dtype"])
    s["logits"] = _held(x, case["dtype"])
    # drafts are drawn from the draft's distribution: the largest logit with Gumbel noise
    noise = -torch.log(-torch.log(torch.rand((b, n - 1, v), generator=g, device=DEVICE).clamp_(1e-12, 1 - 1e-7)))
    real = draft.float() * s["scale"] + noise * (t[:, None, None] if case["mixed"] else t)
    if off is not None:
        real = real.masked_fill(off, -math.inf)
    first = torch.randint(0, v, (b, 1), generator=g, device=DEVICE)
    s["tokens"] = torch.cat([first, real.argmax(-1)], 1) if n > 1 else first
    if case["drawn"]:
        s["draft_logits"] = draft
    # some rows have shorter drafts
    short = torch.randint(1, n + 1, (b,), generator=g, device=DEVICE)
    cut = torch.rand(b, generator=g, device=DEVICE) < 0.2
    s["counts"] = torch.where(cut, short, torch.full_like(short, n)).to(torch.int32)
    s["uniforms"] = torch.rand((b, n), generator=g, device=DEVICE)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        import __graft_entry__
        s["ops"] = __graft_entry__.load_package().drafts
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(s):
    case = s["case"]
    kind = case["kind"]
    if not own:
        return {"window": _plain_window, "sample": _plain_sample, "verify": _plain_verify}[kind](s)
    ops = s["ops"]
    if kind == "window":
        return ops.window_attention(s["q"], s["k"], s["v"], s["lengths"], positions=s["positions"], heads=case["heads"],
                                    before=case["before"], after=case["after"], sinks=case["sinks"], **s["scalars"])
    if kind == "sample":
        return list(ops.sample_tokens(s["logits"], s["uniforms"], temperature=s["temperature"], scale=s["scale"],
                                      suppress=s["suppress"]))
    return list(ops.verify_drafts(s["logits"], s["tokens"], s["draft_logits"], s["uniforms"], s["counts"],
                                  temperature=s["temperature"], scale=s["scale"], suppress=s["suppress"]))


def _rshift(x, n):
    """x / 2^n, halves away from zero, modulo 2^32 (x in 32 bits)."""
    return x if n == 0 else (x + (1 << (n - 1)) - (x < 0).to(x.dtype)) >> n


def _wrap(x):
    return ((x + 2 ** 31) & 0xFFFFFFFF) - 2 ** 31


def _inv_sqrt(x, off):
    """The integer inverse square root: the bits of float32(x) give the first guess, two Newton steps (x in 64 bits)."""
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
        t = _wrap(_wrap(_rshift(_wrap(x * y), off)) * y)
        y = _wrap(_rshift(_wrap(y * _wrap((3 << off) - t)), off + 1))
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


def _plain_window(s):
    case, sc = s["case"], s["scalars"]
    b, n, h, d, cap = (case[x] for x in ("batch", "queries", "heads", "head_dim", "cap"))
    dev = s["q"].device
    lengths = torch.full((b,), cap, device=dev) if s["lengths"] is None else s["lengths"].long()
    at = s["positions"]
    at = lengths[:, None] - n + torch.arange(n, device=dev) if at is None else at.long()
    j = torch.arange(cap, device=dev)
    out = torch.empty((b, n, h * d), dtype=torch.int8, device=dev)
    # batch rows at a time, and of one that is too large for that its queries
    rows = max(1, (1 << 26) // (h * cap * n))
    step = max(1, (1 << 26) // (h * cap))
    for r in range(0, b, rows):
        v = s["v"][r:r + rows]
        g = v.shape[0]
        v = v.transpose(3, 4).reshape(g, h, -1, d) if v.dim() == 5 else v.transpose(2, 3)
        v = v[:, :, :cap].double().reshape(g * h, cap, d)
        k = s["k"][r:r + rows].float().reshape(g * h, cap, d).transpose(1, 2).contiguous()
        for i in range(0, n, step):
            q = s["q"][r:r + rows, i:i + step].unflatten(2, (h, d)).transpose(1, 2).float().flatten(0, 1)
            p = at[r:r + rows, i:i + step, None]
            sees = ((j < lengths[r:r + rows, None, None]) & (j <= p + case["after"])
                    & ((j >= p - case["before"]) | (j < case["sinks"])))[:, None]
            # products of up to 128 terms below 2^14 are exact in 32 bits
            score = torch.bmm(q, k).to(torch.int32).unflatten(0, (g, h)) * sc["qk_multiplier"]
            score = _rshift(score, sc["qk_shift"]).clamp_(-32768, 32767)
            top = score.masked_fill(~sees, -32768).amax(-1, keepdim=True)
            e = torch.where(sees, _shift_exp((top + 1 - score) & 0xFFFF, sc["frac_bits"]), 0)
            total = e.sum(-1, keepdim=True)
            o = torch.bmm(e.double().flatten(0, 1), v).long().unflatten(0, (g, h))  # sums pass 2^24
            inv, off = _inv_sqrt(total, sc["rsqrt_offset"]), sc["rsqrt_offset"]
            y = _wrap(_rshift(_wrap(_wrap(o) * inv), off))
            y = _wrap(_rshift(_wrap(y * inv), off))
            y = _rshift(_wrap(y * sc["av_multiplier"]), sc["av_shift"]).clamp(-127, 127).to(torch.int8)
            out[r:r + rows, i:i + step] = y.transpose(1, 2).flatten(2)
    return out


def _hidden(words, v):
    """Truth values of a bit mask's suppressed tokens."""
    i = torch.arange(v, device=words.device)
    return (words[i >> 5] >> (i & 31)) & 1 > 0


def _weights(logits, scale, t, suppress):
    """Weights of rows [..., vocab] at temperatures t ([...] or one), the largest 1; and their exponents. The
    borders between tokens lie closer than 32 bits tell apart: in 64."""
    x = logits.double()
    if suppress is not None:
        x = x.masked_fill(_hidden(suppress, x.shape[-1]), -math.inf)
    t = torch.as_tensor(t, dtype=torch.float64, device=x.device).expand(x.shape[:-1])[..., None]
    d = x - x.amax(-1, keepdim=True)
    a = torch.where(d == -math.inf, d, d * (scale / torch.where(t > 0, t, 1.0)))
    first = torch.zeros_like(d, dtype=torch.bool).scatter_(-1, (d == 0).long().argmax(-1, keepdim=True), True)
    a = torch.where(t > 0, a, torch.where(first, 0.0, -math.inf))
    return torch.exp(a), a


def _pick(w, u):
    """The least index whose running sum of weights [rows, vocab] passes u times their sum."""
    run = w.cumsum(-1)
    some = w > 0
    last = w.shape[-1] - 1 - some.flip(-1).to(torch.uint8).argmax(-1)
    return torch.minimum((run <= u.double()[:, None] * run[:, -1:]).sum(-1), last)


def _plain_sample(s):
    w, a = _weights(s["logits"], s["scale"], s["temperature"], s["suppress"])
    tok = _pick(w, s["uniforms"])
    return [tok, (a.gather(1, tok[:, None])[:, 0] - torch.log(w.sum(-1))).float()]


def _plain_verify(s):
    b, n = s["tokens"].shape
    dev = s["tokens"].device
    t = s["temperature"]
    t = t[:, None] if isinstance(t, torch.Tensor) else t
    rows = torch.arange(b, device=dev)
    w, _ = _weights(s["logits"], s["scale"], t, s["suppress"])
    p = w / w.sum(-1, keepdim=True)
    drafts = s["tokens"][:, 1:, None]
    if s["draft_logits"] is not None:
        w, _ = _weights(s["draft_logits"], s["scale"], t, s["suppress"])
        q = w / w.sum(-1, keepdim=True)
    else:
        q = torch.zeros_like(p[:, 1:]).scatter_(2, drafts, 1.0)
    px, qx = p[:, :-1].gather(2, drafts)[..., 0], q.gather(2, drafts)[..., 0]
    counts = s["counts"].long()
    ok = (s["uniforms"][:, :-1].double() * qx < px) & (torch.arange(1, n, device=dev) < counts[:, None])
    taken = ok.long().cumprod(1).sum(1)
    at = p[rows, taken]
    if n > 1:
        less = torch.where((taken < counts - 1)[:, None], q[rows, taken.clamp(max=n - 2)], 0.0)
        rest = (at - less).clamp(min=0)
        at = torch.where(rest.sum(-1, keepdim=True) > 0, rest, at)
    nxt = _pick(at, s["uniforms"][:, -1])
    i = torch.arange(n, device=dev)
    choice = torch.cat([s["tokens"][:, 1:], nxt[:, None]], 1)
    choice = torch.where(i < taken[:, None], choice, torch.where(i == taken[:, None], nxt[:, None], -1))
    return [choice, taken.to(torch.int32), nxt]


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = _inputs(case, seed)
    return {"window": _exact_window, "sample": _exact_sample, "verify": _exact_verify}[case["kind"]](case, s)


def _exact_window(case, s):
    # head by head, over the keys that a row has, its probabilities from a table of all 65536 differences
    b, n, h, d, cap = (case[x] for x in ("batch", "queries", "heads", "head_dim", "cap"))
    if b * h * n * cap > 4e10:
        return None
    sc, f = s["scalars"], s["scalars"]["frac_bits"]
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
        ln = cap if s["lengths"] is None else int(s["lengths"][i])
        if ln == 0:
            continue
        pos = range(ln - n, ln) if s["positions"] is None else s["positions"][i].tolist()
        # key borders of each query: from its window's start, up to its end, and the first ones below that
        end = torch.tensor([max(0, min(ln, x + case["after"] + 1)) for x in pos], device=DEVICE)[:, None]
        start = torch.tensor([max(0, x - case["before"]) for x in pos], device=DEVICE)[:, None]
        key = torch.arange(ln, device=DEVICE)
        unseen = (key >= end) | ((key < start) & (key >= case["sinks"]))
        v = s["v"][i]  # [heads, quads, head_dim, 4] or [heads, head_dim, positions]
        v = v.permute(0, 2, 1, 3).reshape(h, d, -1).transpose(1, 2) if v.dim() == 4 else v.transpose(1, 2)
        for g in range(h):
            q = s["q"][i, :, g * d:(g + 1) * d].double()
            score = shr((q @ s["k"][i, g, :ln].double().T.contiguous()).long() * sc["qk_multiplier"], sc["qk_shift"])
            score = score.clamp_(-32768, 32767)
            best = score.masked_fill(unseen, -32768).amax(-1, keepdim=True)
            p = table[(best + 1 - score) % 65536].masked_fill_(unseen, 0)
            o, total = (p @ v[g, :ln].double()).long(), p.sum(-1, keepdim=True).long()
            inv = _inv_sqrt_host(total, sc["rsqrt_offset"])
            y = shr(_wrap(o * inv), sc["rsqrt_offset"])
            y = shr(_wrap(y * inv), sc["rsqrt_offset"])
            out[i, :, g * d:(g + 1) * d] = shr(_wrap(y * sc["av_multiplier"]), sc["av_shift"]).clamp(-127, 127)
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


def _logprob(case, s, name, row, t):
    """Log-probabilities [rows, vocab] of a row's logits at temperature t."""
    x = s[name][row].double() * s["scale"]
    if s["suppress"] is not None:
        bits = [(w >> j) & 1 for w in s["suppress"].tolist() for j in range(32)][:case["vocab"]]
        x[..., torch.tensor(bits, device=DEVICE) == 1] = -math.inf
    if t <= 0:
        best = x.amax(-1, keepdim=True) == x
        return torch.where(best & (best.cumsum(-1) == 1), 0.0, -math.inf)
    return torch.log_softmax(x / t, -1)


def _reach(p, u):
    """The first token whose distribution function passes u, of probabilities [vocab]."""
    f = p.cumsum(0)
    return min(int(torch.searchsorted(f, f[-1:] * u, right=True)), int(p.nonzero()[-1]))


def _temperatures(s, rows):
    t = s["temperature"]
    return t.tolist() if isinstance(t, torch.Tensor) else [t] * rows


def _exact_sample(case, s):
    tok, lp = [], []
    u = s["uniforms"].tolist()
    t = _temperatures(s, case["rows"])
    by = {}  # rows of one temperature at a time
    for r, x in enumerate(t):
        by.setdefault(x, []).append(r)
    tok, lp = torch.zeros(case["rows"], dtype=torch.int64), torch.zeros(case["rows"], dtype=torch.float64)
    for x, rows in by.items():
        for at in range(0, len(rows), 64):
            some = rows[at:at + 64]
            l = _logprob(case, s, "logits", torch.tensor(some, device=DEVICE), x)
            for r, row in zip(some, l):
                tok[r] = _reach(row.exp(), u[r])
                lp[r] = row[int(tok[r])]
    return [tok, lp]


def _exact_verify(case, s):
    b, n = case["batch"], case["nodes"]
    t = _temperatures(s, b)
    tokens, counts, u = s["tokens"].tolist(), s["counts"].tolist(), s["uniforms"].tolist()
    choices, taken, nxt = [], [], []
    for r in range(b):
        p = _logprob(case, s, "logits", r, t[r])
        q = None if s["draft_logits"] is None else _logprob(case, s, "draft_logits", r, t[r])
        a = 0
        while a < counts[r] - 1:
            x = tokens[r][a + 1]
            qx = 1.0 if q is None else math.exp(float(q[a, x]))
            if not u[r][a] * qx < math.exp(float(p[a, x])):
                break
            a += 1
        left = p[a].exp()
        if a < counts[r] - 1:
            if q is None:
                left[tokens[r][a + 1]] = 0.0
            else:
                left = torch.where(p[a] > q[a], left - q[a].exp(), 0.0)
            if float(left.sum()) <= 0:
                left = p[a].exp()
        got = _reach(left, u[r][n - 1])
        choices.append(tokens[r][1:a + 1] + [got] + [-1] * (n - 1 - a))
        taken.append(a)
        nxt.append(got)
    return [torch.tensor(choices, dtype=torch.int64), torch.tensor(taken, dtype=torch.int32),
            torch.tensor(nxt, dtype=torch.int64)]
