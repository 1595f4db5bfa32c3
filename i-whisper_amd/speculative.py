"""Drafted tokens: several of them per row verified in one decoder pass, and tokens scored.

The reference decodes one token per row and step (decoding.py:684-712). Here a
row may bring a tree of up to 64 drafted tokens (of a smaller model, of an
earlier window, of a beam); one pass through the decoder gives the model's
choice after each of them, and the longest path of drafts that the model
would have chosen itself is accepted. Greedy decoding over integer kernels is
reproducible bit for bit, so the tokens are those of ``greedy_decode``.

* ``tree_plan``       which node sees which, and each node's position
* ``tree_attention``  the nodes' attention over the int8 KV caches and the tree
* ``TreeCaches``      accepts a path: K and V of its nodes enter every layer's cache
* ``token_logprobs``  log-probabilities of given tokens, entropy, best alternatives
* ``TreeDecoder``     the pass itself, over a DecoderRunner's model and caches

Node 0 of a row's tree is its last chosen token, whose keys and values are not
in the caches yet; node i hangs on node ``parents[b, i] < i``. Work is queued
on the current stream of the tensors' device and reads nothing back, so every
call can be captured into a graph. Wrong dtypes, shapes and layouts raise
RuntimeError.
"""
from __future__ import annotations

import ctypes
import struct
from typing import NamedTuple, Optional, Sequence

import torch

from . import _lib
from .runtime import DecoderRunner, _ln, _lin8, _lin32_res, _mlp_gelu

Tensor = torch.Tensor

MAX_NODES = 64
MAX_TOP = 32
_LOGIT_TYPES = {torch.int8: 0, torch.float32: 1, torch.bfloat16: 2, torch.float16: 3}
_I8, _I32, _I64 = torch.int8, torch.int32, torch.int64
_ATTENTION_ARGS = struct.Struct("37q")  # iw_attention_tree_args
_CACHES = struct.Struct("21q")          # iw_tree_caches


def _launch(dev: int, name: str, *args) -> None:
    """Call an entry point on the current stream of device ``dev``, the tensors'."""
    if dev == torch._C._cuda_getDevice():
        _lib.call(name, *args, torch._C._cuda_getCurrentRawStream(dev))
    else:
        with torch.cuda.device(dev):
            _lib.call(name, *args, _lib.stream())


# A call's tensors are looked over in one expression; only where that fails are
# they taken one by one, for the message.

def _check(t: Tensor, dtype: torch.dtype, shape: Sequence[int], name: str, dev: Optional[int] = None,
           contiguous: bool = True) -> None:
    if not isinstance(t, torch.Tensor):
        raise RuntimeError(f"{name} must be a tensor")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a GPU tensor, got device {t.device}")
    if t.dtype != dtype:
        raise RuntimeError(f"{name} must be {str(dtype).replace('torch.', '')}, got {t.dtype}")
    if t.shape != tuple(shape):
        raise RuntimeError(f"{name} must have the shape {tuple(shape)}, got {tuple(t.shape)}")
    if dev is not None and t.get_device() != dev:
        raise RuntimeError(f"{name} is on {t.device}, the other tensors on device {dev}")
    if contiguous and not t.is_contiguous():
        raise RuntimeError(f"{name} must be contiguous")


def _is(t: Optional[Tensor], dtype: torch.dtype, shape: Sequence[int], dev: int) -> bool:
    """Whether ``_check`` has nothing to say."""
    return (isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == shape and t.get_device() == dev
            and t.is_contiguous())


def _ptr(t: Optional[Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _pack(layout: struct.Struct, *values) -> bytes:
    try:
        return layout.pack(*values)
    except struct.error as e:
        raise RuntimeError(f"sizes and scalars must be whole numbers of 64 bits: {e}") from None


def _rows_strides(t: Tensor, shape, name: str, dev: int):
    """(batch, node) strides of an int8 [B, N, H * D] operand with contiguous rows."""
    if not (isinstance(t, torch.Tensor) and t.dtype is _I8 and t.shape == shape and t.get_device() == dev):
        _check(t, _I8, shape, name, dev, contiguous=False)
    sb, st, sc = t.stride()
    if sc != 1:
        raise RuntimeError(f"the rows of {name} must be contiguous")
    return (sb if shape[0] > 1 else 0), (st if shape[1] > 1 else 0)


def _cache_strides(k: Tensor, v: Tensor, B: int, H: int, D: int, dev: int):
    """Positions and strides (k_sb, k_sh, k_st), (v_sb, v_sh, v_sd, v_sq) of a layer's caches: K
    [B, H, T, D], V in key quads [B, H, ceil(T / 4), D, 4] or transposed [B, H, D, round_up(T, 16)]."""
    if not isinstance(k, torch.Tensor) or k.dim() != 4:
        raise RuntimeError("k_cache must be [batch, heads, positions, head_dim]")
    T = k.shape[2]
    if not (k.dtype is _I8 and k.shape == (B, H, T, D) and k.get_device() == dev):
        _check(k, _I8, (B, H, T, D), "k_cache", dev, contiguous=False)
    if not isinstance(v, torch.Tensor) or v.dim() not in (4, 5):
        raise RuntimeError("v_cache must be key quads [batch, heads, quads, head_dim, 4] or transposed "
                           "[batch, heads, head_dim, positions]")
    vs, last = v.stride(), v.shape[2 if v.dim() == 5 else 3]
    want = (B, H, last, D, 4) if len(vs) == 5 else (B, H, D, last)
    if not (v.dtype is _I8 and v.shape == want and v.get_device() == dev):
        _check(v, _I8, want, "v_cache", dev, contiguous=False)
    if len(vs) == 5:
        if 4 * last < T or vs[4] != 1 or vs[3] != 4:
            raise RuntimeError("v_cache: packed key quads that cover every position of k_cache are needed")
        v_sd, v_sq = 4, (vs[2] if last > 1 else 4 * D)
    else:
        if last < (T + 15) // 16 * 16 or vs[3] != 1:
            raise RuntimeError("v_cache: transposed rows must cover the positions of k_cache rounded up to 16")
        v_sd, v_sq = vs[2], 4
    ks = k.stride()
    if ks[3] != 1:
        raise RuntimeError("the rows of k_cache must be contiguous")
    if B > 1 and H > 1 and T > 1:
        return T, ks[:3], (vs[0], vs[1], v_sd, v_sq)
    return (T, (ks[0] if B > 1 else 0, ks[1] if H > 1 else 0, ks[2] if T > 1 else 0),
            (vs[0] if B > 1 else 0, vs[1] if H > 1 else 0, v_sd, v_sq))


def _tree_shape(t: Tensor, name: str):
    if not isinstance(t, torch.Tensor) or t.dim() != 2 or not 1 <= t.shape[1] <= MAX_NODES:
        raise RuntimeError(f"{name} must be [batch, nodes] with 1 to {MAX_NODES} nodes")
    return t.shape


def _node_shape(t: Tensor, heads: int, name: str):
    if not isinstance(t, torch.Tensor) or t.dim() != 3 or not 1 <= t.shape[1] <= MAX_NODES:
        raise RuntimeError(f"{name} must be [batch, nodes, heads * head_dim] with 1 to {MAX_NODES} nodes")
    if heads <= 0 or t.shape[2] % heads:
        raise RuntimeError(f"{name}.size(2) must be a multiple of heads")
    return t.shape


class TreePlan(NamedTuple):
    visible: Tensor    # int64 [B, N]: bit j of a node's word = it sees node j
    positions: Tensor  # int32 [B, N]: the row's length plus the node's depth


def tree_plan(parents: Tensor, counts: Optional[Tensor] = None, *, lengths: Optional[Tensor] = None,
              max_positions: int = 2 ** 31 - 1) -> TreePlan:
    """Which nodes a node sees (itself and its ancestors) and its position.

    ``parents`` int32 [B, N] (a parent outside [0, i) makes node i a root);
    ``counts`` int32 [B]: nodes in use, the others see nothing and sit at the
    row's length; ``lengths`` int32 [B]: cached tokens. Positions stay below
    ``max_positions``."""
    B, N = _tree_shape(parents, "parents")
    if not 1 <= max_positions < 2 ** 31:
        raise RuntimeError("max_positions must be in [1, 2^31)")
    dev = parents.get_device()
    if not (dev >= 0 and _is(parents, _I32, (B, N), dev) and (counts is None or _is(counts, _I32, (B,), dev))
            and (lengths is None or _is(lengths, _I32, (B,), dev))):
        _check(parents, _I32, (B, N), "parents")
        for t, name in ((counts, "counts"), (lengths, "lengths")):
            if t is not None:
                _check(t, _I32, (B,), name, dev)
    positions = torch.empty_like(parents)
    visible = torch.empty_like(parents, dtype=_I64)
    _launch(dev, "iw_tree_plan", parents.data_ptr(), N, _ptr(counts), _ptr(lengths), B, N, max_positions,
            visible.data_ptr(), positions.data_ptr())
    return TreePlan(visible, positions)


def tree_attention(q: Tensor, k_new: Tensor, v_new: Tensor, k_cache: Tensor, v_cache: Tensor, lengths: Tensor,
                   visible: Tensor, counts: Optional[Tensor] = None, *, heads: int, qk_multiplier: int,
                   qk_shift: int, frac_bits: int, av_multiplier: int, av_shift: int, rsqrt_offset: int = 16,
                   out: Optional[Tensor] = None) -> Tensor:
    """Integer attention (model_int.py:774-1040) of each row's nodes over its first ``lengths[b]``
    cached keys and the nodes of ``visible`` (``tree_plan``; [B, N], or [N] for one tree of all rows).

    ``q``, ``k_new``, ``v_new`` int8 [B, N, heads * D], also as columns of one fused projection;
    ``k_cache`` int8 [B, heads, T, D]; ``v_cache`` in key quads [B, heads, ceil(T / 4), D, 4] or transposed
    [B, heads, D, round_up(T, 16)]. D is a multiple of 16 up to 128, strides are multiples of 16.
    Lengths and counts are clamped to T and N on the device. Returns int8 [B, N, heads * D] (``out`` where
    given: ``q`` itself, or memory that K, V, the caches and ``q`` have no part in, other columns of the
    same rows included); nodes past ``counts[b]`` and nodes that see no key give zeros. With one node
    a row it is a decode step over rows of different lengths."""
    shape = _node_shape(q, heads, "q")
    dev = q.get_device()
    B, N, C = shape
    D = C // heads
    q_s = _rows_strides(q, shape, "q", dev)
    kn_s = _rows_strides(k_new, shape, "k_new", dev)
    vn_s = _rows_strides(v_new, shape, "v_new", dev)
    T, k_s, v_s = _cache_strides(k_cache, v_cache, B, heads, D, dev)
    shared = isinstance(visible, torch.Tensor) and visible.dim() == 1
    if not (dev >= 0 and _is(lengths, _I32, (B,), dev) and _is(visible, _I64, (N,) if shared else (B, N), dev)
            and (counts is None or _is(counts, _I32, (B,), dev))):
        _check(q, _I8, shape, "q", contiguous=False)
        _check(lengths, _I32, (B,), "lengths", dev)
        _check(visible, _I64, (N,) if shared else (B, N), "visible", dev)
        if counts is not None:
            _check(counts, _I32, (B,), "counts", dev)
    if out is None:
        out = q.new_empty(shape)
        o_s = (N * C, C)
    else:
        o_s = _rows_strides(out, shape, "out", dev)
    # shorter caches need none
    need = _lib.value("iw_attention_tree_workspace", B, heads, N, D, T) if T >= 1536 else 0
    work = q.new_empty(need, dtype=torch.uint8) if need > 0 else None
    args = _pack(_ATTENTION_ARGS, q.data_ptr(), *q_s, k_new.data_ptr(), *kn_s, v_new.data_ptr(), *vn_s,
                 k_cache.data_ptr(), *k_s, v_cache.data_ptr(), *v_s, lengths.data_ptr(), visible.data_ptr(),
                 0 if shared else N, 0 if counts is None else counts.data_ptr(), out.data_ptr(), *o_s, B, heads, N, D, T,
                 qk_multiplier, qk_shift, frac_bits, av_multiplier, av_shift, rsqrt_offset,
                 0 if work is None else work.data_ptr())
    _launch(dev, "iw_attention_tree", args)
    return out


class TreeAccept(NamedTuple):
    path: Tensor        # int32 [B, N]: the accepted nodes, then -1
    accepted: Tensor    # int32 [B]: their number (0 for a row without nodes or room)
    next_token: Tensor  # int64 [B]: the model's choice after the last of them, -1 for none
    lengths: Tensor     # int32 [B]: the rows' lengths with the path cached


def _runs(t: Tensor):
    """The addresses of an int8 tensor's runs of bytes, and their length."""
    dims = sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1)
    length = 1
    while dims and dims[0][0] == length:
        length *= dims.pop(0)[1]
    at = torch.tensor([t.data_ptr()], dtype=torch.int64, device="cpu")
    for s, n in reversed(dims):
        at = (at[:, None] + s * torch.arange(n, device="cpu")).flatten()
    return at, length


def _own_memory(written: Sequence[Tensor], read: Sequence[Tensor]) -> bool:
    """Whether the int8 tensors ``written`` share no byte with one another, with themselves or with
    ``read``. Exact: caches may be parts of one buffer in any order of its dims."""
    spans, layouts = [], {}  # first and last byte; (extent, whether each dim steps over the smaller ones)
    for i, t in enumerate([*written, *read]):
        shape, stride = t.shape, t.stride()
        if (shape, stride) not in layouts:
            end, nested = 1, True
            for s, n in sorted(zip(stride, shape)):
                if n > 1:
                    nested = nested and s >= end
                    end += s * (n - 1)
            layouts[shape, stride] = (0 if 0 in shape else end), nested
        end, nested = layouts[shape, stride]
        if end:
            at = t.data_ptr()
            spans.append((at, at + end, i, nested))
    spans.sort()
    group, end = [], 0
    for lo, hi, i, nested in [*spans, (1 << 62, 1 << 62, -1, True)]:
        if lo >= end:  # none of the tensors before reaches here
            if (len(group) > 1 or group and not group[0][1]) and not _group_apart(
                    [written[j] for j, _ in group if j < len(written)],
                    [read[j - len(written)] for j, _ in group if j >= len(written)]):
                return False
            group = []
        group.append((i, nested))
        end = max(end, hi)
    return True


def _group_apart(written: Sequence[Tensor], read: Sequence[Tensor]) -> bool:
    if not written:
        return True
    runs = [_runs(t) for t in written]
    at = torch.cat([a for a, _ in runs])
    to = torch.cat([a + n for a, n in runs])
    at, order = at.sort()
    to = to[order]
    if bool((to[:-1] > at[1:]).any()):
        return False
    # the last run that starts before a read one ends must end before that one starts
    for a, n in map(_runs, read):
        before = torch.searchsorted(at, a + n) - 1
        if bool(((before >= 0) & (to[before.clamp(min=0)] > a)).any()):
            return False
    return True


class TreeCaches:
    """The layers' caches and the nodes' K and V that a decoder pass leaves for them.

    Lists of one tensor per layer, all with the same shapes and strides:
    ``k_new`` / ``v_new`` int8 [B, N, heads * D] (columns of the projection
    that the pass writes) and the caches as ``tree_attention`` takes them, which
    share no memory with one another or with the nodes' K and V."""

    def __init__(self, k_new: Sequence[Tensor], v_new: Sequence[Tensor], k_cache: Sequence[Tensor],
                 v_cache: Sequence[Tensor], *, heads: int):
        self.tensors = [list(x) for x in (k_new, v_new, k_cache, v_cache)]
        L = len(self.tensors[0])
        if L == 0 or any(len(x) != L for x in self.tensors):
            raise RuntimeError("one k_new, v_new, k_cache and v_cache of each layer are needed")
        kn, vn, k, v = (x[0] for x in self.tensors)
        self.batch, self.nodes, C = shape = _node_shape(kn, heads, "k_new")
        self.device = dev = kn.get_device()
        if dev < 0:
            _check(kn, _I8, shape, "k_new", contiguous=False)
        B, D = self.batch, C // heads
        new = (*_rows_strides(kn, shape, "k_new", dev), *_rows_strides(vn, shape, "v_new", dev))
        self.positions, k_s, v_s = _cache_strides(k, v, B, heads, D, dev)
        for kn_l, vn_l, k_l, v_l in zip(*self.tensors):
            same = (_rows_strides(kn_l, shape, "k_new", dev) + _rows_strides(vn_l, shape, "v_new", dev) == new
                    and _cache_strides(k_l, v_l, B, heads, D, dev) == (self.positions, k_s, v_s))
            if not same:
                raise RuntimeError("the layers' tensors must have the same strides")
        if not _own_memory(self.tensors[2] + self.tensors[3], self.tensors[0] + self.tensors[1]):
            raise RuntimeError("the caches are written: each must be memory of its own")
        self._arrays = [(ctypes.c_void_p * L)(*[t.data_ptr() for t in x]) for x in self.tensors]
        kn_a, vn_a, k_a, v_a = map(ctypes.addressof, self._arrays)
        self._image = _pack(_CACHES, L, B, self.nodes, heads, D, self.positions, kn_a, *new[:2], vn_a, *new[2:], k_a,
                            *k_s, v_a, *v_s)

    def accept(self, tokens: Tensor, parents: Tensor, choice: Tensor, lengths: Tensor,
               counts: Optional[Tensor] = None, *, eot: int = -1) -> TreeAccept:
        """Greedy acceptance: from node 0 on, the first node that hangs on the current one and
        holds the model's choice after it, until there is none, the choice is ``eot`` or the cache is
        full. K and V of the path enter every layer's cache at ``lengths[b]`` and up.

        ``tokens`` int64, ``parents`` int32, ``choice`` int64 (the model's token after each node,
        ``token_logprobs(..., top=1).top_ids``) [B, N]; ``lengths`` and ``counts`` int32 [B]."""
        if not -1 << 63 <= eot < 1 << 63:
            raise RuntimeError("eot must be a token id, or negative for none")
        dev, rows = self.device, (self.batch,)
        shape = (self.batch, self.nodes)
        if not (_is(tokens, _I64, shape, dev) and _is(parents, _I32, shape, dev) and _is(choice, _I64, shape, dev)
                and _is(lengths, _I32, rows, dev) and (counts is None or _is(counts, _I32, rows, dev))):
            _check(tokens, _I64, shape, "tokens", dev)
            _check(parents, _I32, shape, "parents", dev)
            _check(choice, _I64, shape, "choice", dev)
            _check(lengths, _I32, rows, "lengths", dev)
            if counts is not None:
                _check(counts, _I32, rows, "counts", dev)
        path = torch.empty_like(parents)
        accepted = torch.empty_like(lengths)
        after = torch.empty_like(lengths)
        next_token = torch.empty_like(lengths, dtype=_I64)
        _launch(dev, "iw_tree_accept", self._image, tokens.data_ptr(), parents.data_ptr(), choice.data_ptr(),
                _ptr(counts), lengths.data_ptr(), eot, path.data_ptr(), accepted.data_ptr(), next_token.data_ptr(),
                after.data_ptr())
        return TreeAccept(path, accepted, next_token, after)


class TokenLogprobs(NamedTuple):
    logprob: Optional[Tensor]       # float32 [...]: of the targets; None without them
    entropy: Tensor                 # float32 [...]
    top_ids: Optional[Tensor]       # int64 [..., top]; None for top 0
    top_logprobs: Optional[Tensor]  # float32 [..., top]


def token_logprobs(logits: Tensor, targets: Optional[Tensor] = None, *, top: int = 0, scale: float = 1.0,
                   suppress: Optional[Tensor] = None) -> TokenLogprobs:
    """Scores of rows of logits [..., vocab] (int8, float32, bfloat16 or float16), in float32,
    without gradients.

    The real logits are ``logits * scale`` (2^-100 or more; for a decoder's int8 logits
    1 / act_logits_alpha); ``suppress`` is a bit mask of tokens that count as
    -inf (int32 or uint32 words, bit i % 32 of word i // 32, as the runners' filters hold it).
    ``targets`` int64 [...]: tokens whose log-probability is asked for, NaN for one outside
    the vocabulary. ``top`` (at most 32): the most probable tokens in order,
    ties to the lowest index. A row with a NaN or +inf, or without a finite logit, has NaN scores."""
    if not isinstance(logits, torch.Tensor) or not logits.is_cuda or logits.dim() < 1:
        raise RuntimeError("logits must be a GPU tensor [..., vocab]")
    kind = _LOGIT_TYPES.get(logits.dtype)
    if kind is None:
        raise RuntimeError(f"logits must be int8, float32, bfloat16 or float16, got {logits.dtype}")
    dev, lead, V = logits.get_device(), logits.shape[:-1], logits.shape[-1]
    if logits.dim() != 2:
        logits = logits.reshape(-1, V)
    rows = logits.shape[0]
    ld = logits.stride(0) if rows > 1 else V
    if logits.stride(1) != 1 and V > 1 or ld < V:
        logits = logits.contiguous()
        ld = V
    if not 0 <= top <= min(MAX_TOP, V):
        raise RuntimeError(f"top must be in [0, {min(MAX_TOP, V)}]")
    logprob = ids = lps = None
    entropy = logits.new_empty(lead, dtype=torch.float32)
    if targets is not None:
        if not _is(targets, _I64, lead, dev):
            _check(targets, _I64, lead, "targets", dev, contiguous=False)
            targets = targets.contiguous()
        logprob = torch.empty_like(entropy)
    if suppress is not None:
        if not isinstance(suppress, torch.Tensor) or suppress.dtype not in (_I32, torch.uint32):
            raise RuntimeError("suppress must be int32 or uint32 words")
        _check(suppress, suppress.dtype, ((V + 31) // 32,), "suppress", dev)
    if top:
        ids = logits.new_empty((*lead, top), dtype=_I64)
        lps = logits.new_empty((*lead, top), dtype=torch.float32)
    need = _lib.value("iw_token_logprobs_workspace", kind, rows, V, top)
    work = logits.new_empty(need, dtype=torch.uint8) if need > 0 else None
    _launch(dev, "iw_token_logprobs", logits.data_ptr(), kind, rows, V, ld, scale, _ptr(suppress), _ptr(targets),
            _ptr(logprob), entropy.data_ptr(), top, _ptr(ids), _ptr(lps), _ptr(work))
    return TokenLogprobs(logprob, entropy, ids, lps)


class TreeStep(NamedTuple):
    accept: TreeAccept
    scores: TokenLogprobs  # of every node's logits [B, N]: top_ids[..., 0] is the model's choice
    logits: Tensor         # int8 [B, N, vocab]


class TreeDecoder:
    """Decoder passes over trees of drafted tokens, with a DecoderRunner's model and caches.

    Call ``runner.set_audio``, then ``start`` with the prompt, then ``step`` with each
    round of trees. The rows advance by different numbers of tokens (``lengths``, updated in
    place: a captured ``step`` replays on new trees in the same tensors), so the
    runner's own one-token steps are not mixed in before its next ``run``. The runner has
    no logit filters: the choices are the plain first-index argmax."""

    def __init__(self, runner: DecoderRunner, nodes: int):
        if runner.filters is not None:
            raise ValueError("tree decoding takes a runner built without logit filters")
        if not 1 <= nodes <= MAX_NODES:
            raise ValueError(f"a tree has 1 to {MAX_NODES} nodes")
        self.runner, self.nodes = runner, nodes
        r, dec = runner, runner.dec
        B, C, H, D = r.B, r.C, r.H, r.D
        self.M = M = B * nodes
        dev = dec.positional_embedding.device
        i8 = dict(dtype=torch.int8, device=dev)
        # every layer's projection is kept until a path of it is accepted
        self.qkv = [torch.empty((B, nodes, 3 * C), **i8) for _ in dec.blocks]
        v_shape = (B, H, r.tcap16 // 4, D, 4) if r.v_quads else (B, H, D, r.tcap16)
        self.v_cache = [v.view(v_shape) for v in r.v_self]
        self.caches = TreeCaches([t[..., C:2 * C] for t in self.qkv], [t[..., 2 * C:] for t in self.qkv], r.k_self,
                                 self.v_cache, heads=H)
        self.x16 = torch.empty((M, C), dtype=torch.int16, device=dev)
        self.h8 = torch.empty((M, C), **i8)
        self.wv = torch.empty((B, nodes, C), **i8)
        self.qc = torch.empty((M, C), **i8)
        self.f8 = torch.empty((M, 4 * C), **i8)
        self.lengths = torch.zeros(B, dtype=torch.int32, device=dev)

    def start(self, prompt: Tensor) -> Tensor:
        """The prompt step: returns each row's first token [B] (node 0 of its first tree)."""
        r = self.runner
        with torch.cuda.device(self.lengths.device):  # the runner launches on the current device
            r.run(prompt, 1)
        self.lengths.fill_(prompt.shape[1])
        return r.tokens.clone()

    def verify(self, tokens: Tensor, parents: Tensor, counts: Optional[Tensor] = None) -> Tensor:
        """int8 logits [B, N, vocab] after every node; the caches stay as they are."""
        dev, shape = self.lengths.get_device(), (self.runner.B, self.nodes)
        _check(tokens, _I64, shape, "tokens", dev)
        _check(parents, _I32, shape, "parents", dev)
        with torch.cuda.device(dev):  # the runner's parts launch on the current device
            return self._pass(tokens, parents, counts)

    def _pass(self, tokens: Tensor, parents: Tensor, counts: Optional[Tensor]) -> Tensor:
        r, dec, N, M = self.runner, self.runner.dec, self.nodes, self.M
        B, C, H = r.B, r.C, r.H
        dev = self.lengths.get_device()
        plan = tree_plan(parents, counts, lengths=self.lengths, max_positions=dec.n_ctx)
        # unused nodes may hold any value
        emb = dec.token_embedding.weight[tokens.clamp(0, dec.n_vocab - 1)]
        pe = dec.positional_embedding[plan.positions]
        sc0 = dec.scalars()
        x16, h8, wv = self.x16, self.h8, self.wv
        _launch(dev, "iw_add_requant15", emb.data_ptr(), pe.data_ptr(), sc0["m16"].data_ptr(), sc0["s"].data_ptr(),
                x16.data_ptr(), 1, M, C, 1, 1)
        for l, blk in enumerate(dec.blocks):
            sc, s = blk._scalars(), blk.attn._scalars()
            _ln(blk.attn_ln, x16, M, h8)
            qkv = r.self_qkv[l].linear8(h8, M, self.qkv[l])
            tree_attention(qkv[..., :C], qkv[..., C:2 * C], qkv[..., 2 * C:], r.k_self[l], self.v_cache[l],
                           self.lengths, plan.visible, counts, heads=H, qk_multiplier=s["qm"], qk_shift=s["qs"],
                           frac_bits=s["f"], av_multiplier=s["am"], av_shift=s["as_"],
                           rsqrt_offset=blk.attn.rsqrt_offset, out=wv)
            _lin32_res(blk.attn.out, wv.data_ptr(), M, x16, sc["a"])
            _ln(blk.cross_attn_ln, x16, M, h8)
            _lin8(blk.cross_attn.query, h8.data_ptr(), M, self.qc)
            r._cross_attend(blk.cross_attn, l, self.qc.data_ptr(), N * C, C, N, wv, r.cross_tables[l])
            _lin32_res(blk.cross_attn.out, wv.data_ptr(), M, x16, sc["c"])
            _ln(blk.mlp_ln, x16, M, h8)
            _mlp_gelu(blk, h8.data_ptr(), M, self.f8)
            _lin32_res(blk.mlp[2], self.f8.data_ptr(), M, x16, sc["m"])
        _ln(dec.ln, x16, M, h8)
        return dec.classify(h8.view(B, N, C))

    def step(self, tokens: Tensor, parents: Tensor, counts: Optional[Tensor] = None, *, top: int = 1,
             eot: int = -1) -> TreeStep:
        """One round: ``verify``, the choices and their ``top`` alternatives, and the accepted paths."""
        if top < 1:
            raise ValueError("top must be at least 1")
        logits = self.verify(tokens, parents, counts)
        scores = token_logprobs(logits, top=top, scale=self.runner.logit_scale)
        choice = scores.top_ids[..., 0].contiguous()
        got = self.caches.accept(tokens, parents, choice, self.lengths, counts, eot=eot)
        self.lengths.add_(got.accepted)
        return TreeStep(got, scores, logits)
