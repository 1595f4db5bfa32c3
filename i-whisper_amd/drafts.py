"""Sampled decoding, with drafts that the model makes itself.

At a temperature T the reference draws each token from softmax(logits / T), one
per row and step (decoding.py:275-287, the temperatures of its fallback in
transcribe.py). Here the random numbers are given, so a run can be repeated,
and several tokens of a row can be drafted and verified in one decoder pass
without changing their distribution: a draft x drawn from q is accepted with
probability min(1, p(x) / q(x)), else replaced by a token of max(p - q, 0).
Drafts may come from any model, or from this one over a window of the keys: where
the reading of K and V bounds a step such a draft costs less (128 rows of the large
shape with 257 of 1500 audio positions 3.3 ms, a step 5.4), for a row alone as much.

* ``window_attention``  integer attention over the keys around each query's position and a
                        few first ones (also an encoder's local attention)
* ``sample_tokens``     a token of each row of logits, drawn by a given number
* ``verify_drafts``     the drafts of each row accepted or replaced
* ``DraftDecoder``      the three as one loop, over a DecoderRunner's model and caches

Work is queued on the current stream of the tensors' device and reads nothing back,
so every call can be captured into a graph. Wrong dtypes, shapes and layouts
raise RuntimeError.
"""
from __future__ import annotations

import struct
from typing import NamedTuple, Optional, Tuple, Union

import torch

from . import _lib
from .runtime import DecoderRunner, _ln, _lin8, _lin32_res, _mlp_gelu
from .speculative import (_I8, _I32, _I64, _LOGIT_TYPES, MAX_NODES, TreeAccept, TreeCaches, TreeDecoder, _cache_strides,
                          _check, _is, _launch, _pack, _ptr, _rows_strides)

Tensor = torch.Tensor

_F32 = torch.float32
_WINDOW_ARGS = struct.Struct("34q")       # iw_attention_window_args
_SAMPLE_ARGS = struct.Struct("5q2d6q")    # iw_sample_tokens_args
_VERIFY_ARGS = struct.Struct("10q4d10q")  # iw_verify_drafts_args
_FAR = (1 << 31) - 1


def window_attention(q: Tensor, k: Tensor, v: Tensor, lengths: Optional[Tensor] = None, *, heads: int,
                     before: Optional[int], after: Optional[int] = 0, sinks: int = 0, positions: Optional[Tensor] = None,
                     counts: Optional[Tensor] = None, qk_multiplier: int, qk_shift: int, frac_bits: int,
                     av_multiplier: int, av_shift: int, rsqrt_offset: int = 16, out: Optional[Tensor] = None) -> Tensor:
    """Integer attention (model_int.py:774-1040) of each query over the keys around its position.

    The query at position p sees key j of its row's ``lengths[b]`` where ``p - before <= j <= p + after``,
    and of the first ``sinks`` those up to ``p + after`` (None: no bound on that side). ``positions``
    int32 [B, N]; without them the queries are the row's last ones: query i of ``counts[b]`` (or N)
    is at ``lengths[b] - counts[b] + i``.

    ``q`` int8 [B, N, heads * D], also as columns of one fused projection; ``k`` int8 [B, heads, T, D],
    a cache or a view of projected rows; ``v`` in key quads [B, heads, ceil(T / 4), D, 4] or transposed
    [B, heads, D, round_up(T, 16)]; ``lengths`` int32 [B] (None: T). D is a multiple of 16 up to 128,
    strides are multiples of 16. Lengths and counts are clamped to T and N on the device. Returns int8
    [B, N, heads * D] (``out`` where given: ``q`` itself, or memory that ``q``, ``k`` and ``v`` have no
    part in, other columns of the same rows included); queries past ``counts[b]`` and queries that see no
    key give zeros."""
    if not isinstance(q, torch.Tensor) or q.dim() != 3 or heads <= 0 or q.shape[2] % heads:
        raise RuntimeError("q must be [batch, queries, heads * head_dim]")
    B, N, C = shape = q.shape
    D, dev = C // heads, q.get_device()
    q_s = _rows_strides(q, shape, "q", dev)
    T, k_s, v_s = _cache_strides(k, v, B, heads, D, dev)
    if not (dev >= 0 and (lengths is None or _is(lengths, _I32, (B,), dev))
            and (positions is None or _is(positions, _I32, (B, N), dev))
            and (counts is None or _is(counts, _I32, (B,), dev))):
        _check(q, _I8, shape, "q", contiguous=False)
        for t, want, name in ((lengths, (B,), "lengths"), (positions, (B, N), "positions"), (counts, (B,), "counts")):
            if t is not None:
                _check(t, _I32, want, name, dev)
    before = _FAR if before is None else before
    after = _FAR if after is None else after
    if out is None:
        out = q.new_empty(shape)
        o_s = (N * C, C)
    else:
        o_s = _rows_strides(out, shape, "out", dev)
    need = _lib.value("iw_attention_window_workspace", B, heads, N, D, T, before, after, sinks) if T >= 1024 else 0
    work = q.new_empty(need, dtype=torch.uint8) if need > 0 else None
    args = _pack(_WINDOW_ARGS, q.data_ptr(), *q_s, k.data_ptr(), *k_s, v.data_ptr(), *v_s, _ptr(lengths) or 0,
                 _ptr(positions) or 0, N, _ptr(counts) or 0, out.data_ptr(), *o_s, B, heads, N, D, T, before, after,
                 sinks, qk_multiplier, qk_shift, frac_bits, av_multiplier, av_shift, rsqrt_offset, _ptr(work) or 0)
    _launch(dev, "iw_attention_window", args)
    return out


def _logit_type(logits: Tensor, name: str, dims: str) -> int:
    if not isinstance(logits, torch.Tensor) or not logits.is_cuda:
        raise RuntimeError(f"{name} must be a GPU tensor {dims}")
    kind = _LOGIT_TYPES.get(logits.dtype)
    if kind is None:
        raise RuntimeError(f"{name} must be int8, float32, bfloat16 or float16, got {logits.dtype}")
    return kind


def _check_suppress(suppress: Tensor, V: int, dev: int) -> None:
    if not isinstance(suppress, torch.Tensor) or suppress.dtype not in (_I32, torch.uint32):
        raise RuntimeError("suppress must be int32 or uint32 words")
    _check(suppress, suppress.dtype, ((V + 31) // 32,), "suppress", dev)


def _temperature(t: Union[float, Tensor], shape, name: str, dev: int) -> Tuple[float, int]:
    """A temperature of all rows, or the address of the rows' own."""
    if isinstance(t, torch.Tensor):
        if not _is(t, _F32, shape, dev):
            _check(t, _F32, shape, name, dev)
        return 0.0, t.data_ptr()
    return t, 0


class TokenSamples(NamedTuple):
    tokens: Tensor   # int64 [...]
    logprob: Tensor  # float32 [...]: log-probability with which each was drawn


def sample_tokens(logits: Tensor, uniforms: Tensor, *, temperature: Union[float, Tensor] = 1.0, scale: float = 1.0,
                  suppress: Optional[Tensor] = None) -> TokenSamples:
    """A token of each row of logits [..., vocab] (int8, float32, bfloat16 or float16): the first
    whose running sum of softmax(logits * scale / temperature) passes its number of ``uniforms``
    (float32 [...], in [0, 1)).

    ``temperature``: one of all rows, or float32 [...]; 0 takes the first of the largest logits.
    ``suppress`` is a bit mask of tokens that are never drawn (int32 or uint32 words, as
    ``token_logprobs`` takes it). Probabilities are 64-bit. A row with a NaN or +inf, or without a
    finite logit, gives token -1 and a NaN."""
    kind = _logit_type(logits, "logits", "[..., vocab]")
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise RuntimeError("logits must be a GPU tensor [..., vocab]")
    dev, lead, V = logits.get_device(), logits.shape[:-1], logits.shape[-1]
    if logits.dim() != 2:
        logits = logits.reshape(-1, V)
    rows = logits.shape[0]
    ld = logits.stride(0) if rows > 1 else V
    if logits.stride(1) != 1 and V > 1 or ld < V:
        logits = logits.contiguous()
        ld = V
    if not _is(uniforms, _F32, lead, dev):
        _check(uniforms, _F32, lead, "uniforms", dev)
    t, t_rows = _temperature(temperature, lead, "temperature", dev)
    if suppress is not None:
        _check_suppress(suppress, V, dev)
    logprob = torch.empty_like(uniforms)
    tokens = torch.empty_like(uniforms, dtype=_I64)
    need = _lib.value("iw_sample_tokens_workspace", kind, rows, V)
    work = logits.new_empty(max(need, 0), dtype=torch.uint8)
    args = _pack(_SAMPLE_ARGS, logits.data_ptr(), kind, rows, V, ld, scale, t, t_rows, _ptr(suppress) or 0,
                 uniforms.data_ptr(), tokens.data_ptr(), logprob.data_ptr(), work.data_ptr())
    _launch(dev, "iw_sample_tokens", args)
    return TokenSamples(tokens, logprob)


class DraftVerdict(NamedTuple):
    choice: Tensor      # int64 [B, N]: the accepted drafts, the token after them, then -1
    accepted: Tensor    # int32 [B]: the number of drafts accepted (0 .. N - 1)
    next_token: Tensor  # int64 [B]: the token after them, -1 for none

    def nodes(self, counts: Optional[Tensor] = None) -> Tensor:
        """int32 [B]: each row's nodes up to its last accepted draft, the ``counts`` of ``TreeCaches.accept``;
        ``counts`` are those that ``verify_drafts`` was given."""
        taken = self.accepted + 1
        return taken if counts is None else torch.minimum(taken, counts)


def _node_logits(logits: Tensor, shape, name: str, dev: int) -> Tuple[int, int]:
    """(batch, node) strides of logits [B, N, vocab] with contiguous rows."""
    if logits.shape != tuple(shape):
        raise RuntimeError(f"{name} must have the shape {tuple(shape)}, got {tuple(logits.shape)}")
    if logits.get_device() != dev:
        raise RuntimeError(f"{name} is on {logits.device}, the other tensors on device {dev}")
    sb, sn, sv = logits.stride()
    if sv != 1 and shape[2] > 1:
        raise RuntimeError(f"the rows of {name} must be contiguous")
    return sb, sn


def verify_drafts(logits: Tensor, tokens: Tensor, draft_logits: Optional[Tensor], uniforms: Tensor,
                  counts: Optional[Tensor] = None, *, temperature: Union[float, Tensor] = 1.0, scale: float = 1.0,
                  draft_temperature: Union[float, Tensor, None] = None, draft_scale: Optional[float] = None,
                  suppress: Optional[Tensor] = None) -> DraftVerdict:
    """The drafted tokens of each row accepted or replaced, so that the row's tokens are drawn
    from its model's distribution whatever they were drafted from.

    ``tokens`` int64 [B, N]: node 0 is the row's last chosen token, nodes 1 to ``counts[b] - 1`` (int32
    [B], None: N) its drafts in order; N is at most 64. ``logits`` [B, N, vocab] are the model's after
    each node, ``draft_logits`` [B, N - 1, vocab] of the same type those that the drafts were drawn from,
    None where the drafts were certain (of an earlier window, of a table). Draft i + 1 is accepted where
    ``uniforms[b, i] * q(x) < p(x)``; the token after the accepted ones is drawn by ``uniforms[b, N - 1]``
    as ``sample_tokens`` does, from max(p - q, 0) where a draft was refused and else from p.

    ``temperature`` (one, or float32 [B]; 0: the first of the largest logits) and ``scale`` are those of
    ``sample_tokens``, for the drafts ``draft_temperature`` and ``draft_scale`` (None: the same);
    ``suppress`` counts for both. A row whose next token has no distribution (NaN, +inf, no finite logit)
    gives -1, and so does one without nodes; a draft whose logits have none is refused, and the token drawn
    from p may be that draft again. So ``TreeCaches.accept`` takes ``choice`` for the chain of the nodes
    together with ``nodes(counts)`` of the verdict, which end where the accepted drafts do."""
    kind = _logit_type(logits, "logits", "[batch, nodes, vocab]")
    if logits.dim() != 3 or not 1 <= logits.shape[1] <= MAX_NODES or logits.shape[2] < 1:
        raise RuntimeError(f"logits must be [batch, nodes, vocab] with 1 to {MAX_NODES} nodes")
    dev = logits.get_device()
    B, N, V = logits.shape
    sb, sn = _node_logits(logits, (B, N, V), "logits", dev)
    d_sb = d_sn = 0
    if draft_logits is not None:
        if _logit_type(draft_logits, "draft_logits", "[batch, nodes - 1, vocab]") != kind:
            raise RuntimeError(f"draft_logits must be of the logits' type {logits.dtype}, got {draft_logits.dtype}")
        d_sb, d_sn = _node_logits(draft_logits, (B, N - 1, V), "draft_logits", dev)
    if not (_is(tokens, _I64, (B, N), dev) and _is(uniforms, _F32, (B, N), dev)
            and (counts is None or _is(counts, _I32, (B,), dev))):
        _check(tokens, _I64, (B, N), "tokens", dev)
        _check(uniforms, _F32, (B, N), "uniforms", dev)
        if counts is not None:
            _check(counts, _I32, (B,), "counts", dev)
    t, t_rows = _temperature(temperature, (B,), "temperature", dev)
    if draft_temperature is None:
        dt, dt_rows = t, t_rows
    else:
        dt, dt_rows = _temperature(draft_temperature, (B,), "draft_temperature", dev)
    if suppress is not None:
        _check_suppress(suppress, V, dev)
    choice = torch.empty_like(tokens)
    accepted = tokens.new_empty(B, dtype=_I32)
    next_token = tokens.new_empty(B)
    need = _lib.value("iw_verify_drafts_workspace", kind, B, N, V, draft_logits is not None)
    work = logits.new_empty(max(need, 0), dtype=torch.uint8)
    args = _pack(_VERIFY_ARGS, logits.data_ptr(), sb, sn, _ptr(draft_logits) or 0, d_sb, d_sn, kind, B, N, V, scale, t,
                 scale if draft_scale is None else draft_scale, dt, t_rows, dt_rows, _ptr(suppress) or 0,
                 tokens.data_ptr(), _ptr(counts) or 0, uniforms.data_ptr(), choice.data_ptr(), accepted.data_ptr(),
                 next_token.data_ptr(), work.data_ptr())
    _launch(dev, "iw_verify_drafts", args)
    return DraftVerdict(choice, accepted, next_token)


class DraftStep(NamedTuple):
    tokens: Tensor         # int64 [B, N]: the row's last token and its drafts
    verdict: DraftVerdict
    accept: TreeAccept     # as of a chain: accepted counts node 0, next_token is the last token of the next step


class DraftDecoder:
    """Sampled decoding with drafts of the model itself, over a DecoderRunner's model and caches.

    A step drafts ``nodes - 1`` tokens one after the other with attention over a window of the keys,
    then verifies them in one pass over all keys; the rows advance by different numbers of tokens.
    ``window`` and ``sinks``: cached tokens that a draft sees (None: all). ``audio``: with ``frames``
    given to a step, a draft's cross-attention sees that many audio positions before and after the
    row's frame and the first ``audio_sinks`` (None: all audio).

    Call ``runner.set_audio``, then ``start`` with the prompt, then ``step``. With one node a step is
    plain sampling. ``uniforms`` are float32 in [0, 1), the only source of chance. The runner has no logit
    filters; ``suppress`` tokens are never drawn."""

    def __init__(self, runner: DecoderRunner, nodes: int, *, window: Optional[int] = None, sinks: int = 4,
                 audio: Optional[int] = None, audio_sinks: int = 0, suppress: Optional[Tensor] = None):
        for name, x in (("window", window), ("sinks", sinks), ("audio", audio), ("audio_sinks", audio_sinks)):
            if x is not None and not 0 <= x <= _FAR:
                raise ValueError(f"{name} must be a number of keys")
        self.tree = TreeDecoder(runner, nodes)
        self.runner, self.nodes = runner, nodes
        self.window, self.sinks, self.audio, self.audio_sinks = window, sinks, audio, audio_sinks
        r, dec = runner, runner.dec
        B, C = r.B, r.C
        dev = self.tree.lengths.device
        self.suppress = suppress
        if suppress is not None:
            _check_suppress(suppress, dec.n_vocab, dev.index)
        i8 = dict(dtype=_I8, device=dev)
        # one draft's projection, appended to a layer's caches before its attention
        self.qkv = torch.empty((B, 1, 3 * C), **i8)
        self.appends = [TreeCaches([self.qkv[..., C:2 * C]], [self.qkv[..., 2 * C:]], [k], [v], heads=r.H)
                        for k, v in zip(r.k_self, self.tree.v_cache)]
        self.h8 = torch.empty((B, C), **i8)
        self.x16 = torch.empty((B, C), dtype=torch.int16, device=dev)
        self.wv = torch.empty((B, 1, C), **i8)
        self.qc = torch.empty((B, 1, C), **i8)
        self.f8 = torch.empty((B, 4 * C), **i8)
        self.draft_logits = torch.empty((nodes - 1, B, dec.n_vocab), **i8)
        self.tokens = torch.zeros((B, nodes), dtype=_I64, device=dev)
        self.parents = (torch.arange(nodes, dtype=_I32, device=dev) - 1).repeat(B, 1)
        self._root = torch.full((B, 1), -1, dtype=_I32, device=dev)

    @property
    def lengths(self) -> Tensor:
        """Cached tokens of each row, int32 [B]."""
        return self.tree.lengths

    def start(self, prompt: Tensor, uniforms: Tensor, temperature: Union[float, Tensor] = 1.0) -> Tensor:
        """The prompt step: returns each row's first token [B], drawn by ``uniforms`` float32 [B]."""
        self.tree.start(prompt)
        return sample_tokens(self.runner.logits, uniforms, temperature=temperature, scale=self.runner.logit_scale,
                             suppress=self.suppress).tokens

    def draft(self, last: Tensor, uniforms: Tensor, temperature: Union[float, Tensor] = 1.0,
              frames: Optional[Tensor] = None) -> Tensor:
        """``last`` int64 [B] and ``nodes - 1`` tokens drafted after it, int64 [B, nodes]; ``uniforms`` float32
        [B, nodes - 1]; ``frames`` int32 [B]: the audio position where each row is. The drafts' logits are left in
        ``draft_logits``, their K and V in the caches behind the rows' lengths."""
        dev, B = self.lengths.get_device(), self.runner.B
        _check(last, _I64, (B,), "last", dev, contiguous=False)
        _check(uniforms, _F32, (B, self.nodes - 1), "uniforms", dev, contiguous=False)
        if frames is not None:
            _check(frames, _I32, (B,), "frames", dev)
        with torch.cuda.device(dev):  # the runner's parts launch on the current device
            self.tokens[:, 0] = last
            for i in range(self.nodes - 1):
                self._one(i, frames)
                got = sample_tokens(self.draft_logits[i], uniforms[:, i].contiguous(), temperature=temperature,
                                    scale=self.runner.logit_scale, suppress=self.suppress)
                self.tokens[:, i + 1] = got.tokens
        return self.tokens

    def _one(self, i: int, frames: Optional[Tensor]) -> None:
        """The decoder's pass over draft i, its logits into ``draft_logits[i]``."""
        r, dec = self.runner, self.runner.dec
        B, C, H = r.B, r.C, r.H
        dev = self.lengths.get_device()
        at = self.lengths + i
        token = self.tokens[:, i:i + 1].contiguous()
        emb = dec.token_embedding.weight[token[:, 0].clamp(0, dec.n_vocab - 1)]
        pe = dec.positional_embedding[at.clamp(max=dec.n_ctx - 1)]
        sc0 = dec.scalars()
        x16, h8, wv, qkv = self.x16, self.h8, self.wv, self.qkv
        _launch(dev, "iw_add_requant15", emb.data_ptr(), pe.data_ptr(), sc0["m16"].data_ptr(), sc0["s"].data_ptr(),
                x16.data_ptr(), 1, B, C, 1, 1)
        after = at + 1
        for l, blk in enumerate(dec.blocks):
            sc = blk._scalars()
            _ln(blk.attn_ln, x16, B, h8)
            r.self_qkv[l].linear8(h8, B, qkv)
            self.appends[l].accept(token, self._root, token, at)
            self._attend(blk.attn, qkv[..., :C], r.k_self[l], self.tree.v_cache[l], after, None, self.window, 0, self.sinks)
            _lin32_res(blk.attn.out, wv.data_ptr(), B, x16, sc["a"])
            _ln(blk.cross_attn_ln, x16, B, h8)
            _lin8(blk.cross_attn.query, h8.data_ptr(), B, self.qc)
            if frames is None or self.audio is None:
                r._cross_attend(blk.cross_attn, l, self.qc.data_ptr(), C, C, 1, wv, None)
            else:
                self._attend(blk.cross_attn, self.qc, r.k_cross[l], r.vt_cross[l], None, frames.view(B, 1), self.audio,
                             self.audio, self.audio_sinks)
            _lin32_res(blk.cross_attn.out, wv.data_ptr(), B, x16, sc["c"])
            _ln(blk.mlp_ln, x16, B, h8)
            _mlp_gelu(blk, h8.data_ptr(), B, self.f8)
            _lin32_res(blk.mlp[2], self.f8.data_ptr(), B, x16, sc["m"])
        _ln(dec.ln, x16, B, h8)
        _launch(dev, "iw_classifier", h8.data_ptr(), dec.token_embedding.weight.data_ptr(), sc0["cm"], sc0["cs"],
                self.draft_logits[i].data_ptr(), B, C, dec.n_vocab)

    def _attend(self, att, q, k, v, lengths, positions, before, after, sinks) -> None:
        s = att._scalars()
        window_attention(q, k, v, lengths, heads=self.runner.H, before=before, after=after, sinks=sinks,
                         positions=positions, qk_multiplier=s["qm"], qk_shift=s["qs"], frac_bits=s["f"],
                         av_multiplier=s["am"], av_shift=s["as_"], rsqrt_offset=att.rsqrt_offset, out=self.wv)

    def step(self, last: Tensor, uniforms: Tensor, temperature: Union[float, Tensor] = 1.0, *,
             frames: Optional[Tensor] = None, eot: int = -1) -> DraftStep:
        """Drafts after ``last`` int64 [B], one verifying pass, and the accepted tokens' K and V in the caches.

        ``uniforms`` float32 [B, 2 * nodes - 1]: those that draw the drafts, then those that verify them. The row's
        new tokens are the first ``accept.accepted[b]`` of ``verdict.choice[b]`` (an ``eot`` ends them, a full
        cache too), the last of which is ``accept.next_token[b]``."""
        n, dev = self.nodes, self.lengths.get_device()
        _check(uniforms, _F32, (self.runner.B, 2 * n - 1), "uniforms", dev, contiguous=False)
        tokens = self.draft(last, uniforms[:, :n - 1], temperature, frames)
        logits = self.tree.verify(tokens, self.parents)
        verdict = verify_drafts(logits, tokens, self.draft_logits.transpose(0, 1) if n > 1 else None,
                                uniforms[:, n - 1:].contiguous(), temperature=temperature, scale=self.runner.logit_scale,
                                suppress=self.suppress)
        got = self.tree.caches.accept(tokens, self.parents, verdict.choice, self.lengths, verdict.nodes(), eot=eot)
        self.lengths.add_(got.accepted)
        return DraftStep(tokens.clone(), verdict, got)
