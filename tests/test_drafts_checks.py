"""Refusals of the operators of sampled decoding with drafts, before any device work: the
C entry points with sizes, alignments and overlaps they do not take, and the Python layer with
tensors that are not what it needs. No GPU."""
import struct
from types import SimpleNamespace

import pytest
import torch

P = 1 << 20  # any address will do: a refused call reads nothing

WINDOW = dict(q=P, q_sb=1024, q_st=128, k=P << 4, k_sb=8192, k_sh=4096, k_st=64, v=P << 5, v_sb=8192, v_sh=4096, v_sd=4, v_sq=256,
              lengths=P, positions=P, pos_sb=8, counts=None, out=P << 3, o_sb=1024, o_st=128, batch=2, heads=2, queries=8,
              D=64, cap=64, before=9, after=0, sinks=2, qm=3, qs=4, f=8, am=3, as_=4, off=16, work=None)
SAMPLE = dict(x=P, type=0, rows=2, cols=100, ld=100, scale=1.0, t=1.0, ts=None, suppress=None, u=P, tokens=P, lp=P, work=P)
VERIFY = dict(x=P, sb=400, sn=100, d=P, d_sb=300, d_sn=100, type=0, batch=2, nodes=4, cols=100, scale=1.0, t=1.0,
              d_scale=1.0, dt=1.0, ts=None, dts=None, suppress=None, tokens=P, counts=None, u=P, choice=P, accepted=P, next=P,
              work=P)
FORMS = {"iw_attention_window": "34q", "iw_sample_tokens": "5q2d6q", "iw_verify_drafts": "10q4d10q"}


def call(iw, name, args):
    lib = iw._lib.load()
    image = struct.pack(FORMS[name], *[0 if x is None else x for x in args.values()])
    return getattr(lib, name)(image, None), lib.iw_last_error().decode()


def refused(iw, name, args, change, what):
    rc, msg = call(iw, name, {**args, **change})
    assert rc == -1 and what in msg, msg


@pytest.mark.parametrize("change,what", [
    (dict(f=0), "frac_bits"), (dict(f=14), "frac_bits"), (dict(off=30), "rsqrt_offset"), (dict(off=-1), "rsqrt_offset"),
    (dict(qm=256), "uint8"), (dict(am=-1), "uint8"), (dict(qs=128), "int8"), (dict(as_=-129), "int8"),
    (dict(D=8), "head_dim"), (dict(D=144), "head_dim"), (dict(D=0), "head_dim"), (dict(heads=0), "head_dim"),
    (dict(heads=4097), "head_dim"), (dict(cap=0), "positions"), (dict(cap=1 << 24), "positions"),
    (dict(v_sd=8), "quads"), (dict(v_sq=128), "quads"), (dict(v_sq=4, v_sd=48), "transposed"),
    (dict(queries=-1), "queries"), (dict(queries=(1 << 24) + 1), "queries"), (dict(batch=-1), "shape"),
    (dict(batch=(1 << 21) + 1), "shape"), (dict(pos_sb=-8), "shape"), (dict(batch=1 << 20, queries=1 << 20), "shape"),
    (dict(before=-1), "before"), (dict(after=-1), "before"), (dict(sinks=-1), "before"), (dict(before=1 << 31), "before"),
    (dict(after=1 << 31), "before"), (dict(sinks=1 << 31), "before"), (dict(q=None), "null"), (dict(k=None), "null"),
    (dict(v=None), "null"), (dict(out=None), "null"), (dict(q=P + 8), "16-byte"), (dict(k=P + 1), "16-byte"),
    (dict(out=(P << 3) + 4), "16-byte"), (dict(q_st=136), "16-byte"), (dict(k_sh=4100), "16-byte"), (dict(v_sq=264), "16-byte"),
    (dict(o_st=132), "16-byte"), (dict(k_st=1 << 25), "2^25"), (dict(v_sq=1 << 25), "2^25"), (dict(k_st=-64), "2^25"),
    (dict(o_st=64), "rows of out"), (dict(o_sb=512), "rows of out"), (dict(out=P + 64), "overlap q"),
    (dict(out=P << 4), "keys or values"), (dict(out=P << 5), "keys or values"), (dict(out=(P << 4) + 8192), "keys or values")])
def test_window_refusals(iw, change, what):
    refused(iw, "iw_attention_window", WINDOW, change, what)


def test_window_out_beside_the_keys_of_rows(iw):
    """Keys as columns of a projection's rows: out may be other columns of them, or of q, but not theirs."""
    rows = dict(WINDOW, q_sb=384 * 64, q_st=384, k=P + 128, k_sb=384 * 64, k_sh=64, k_st=384, queries=64, o_sb=384 * 64,
                o_st=384)
    for out in (P + 128, P + 64, P + 192):
        refused(iw, "iw_attention_window", rows, dict(out=out), "overlap")
    refused(iw, "iw_attention_window", dict(rows, k_sh=4096), dict(out=P + 256), "keys or values")


@pytest.mark.parametrize("change,what", [
    (dict(type=4), "int8"), (dict(type=-1), "int8"), (dict(rows=-1), "shape"), (dict(rows=(1 << 22) + 1), "shape"), (dict(cols=0), "shape"),
    (dict(cols=1 << 23, ld=1 << 23), "shape"), (dict(ld=99), "shape"), (dict(type=1, x=P + 2), "aligned"),
    (dict(type=2, x=P + 1), "aligned"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(t=-0.1), "temperature"), (dict(t=float("nan")), "temperature"),
    (dict(t=float("inf")), "temperature"), (dict(x=None), "null"), (dict(u=None), "null"), (dict(tokens=None), "null"),
    (dict(work=None), "workspace"), (dict(work=P + 8), "workspace")])
def test_sample_refusals(iw, change, what):
    refused(iw, "iw_sample_tokens", SAMPLE, change, what)


@pytest.mark.parametrize("change,what", [
    (dict(type=4), "int8"), (dict(batch=-1), "shape"), (dict(batch=(1 << 20) + 1), "rows"), (dict(cols=0), "shape"),
    (dict(cols=1 << 23), "shape"), (dict(nodes=0), "64 nodes"), (dict(nodes=65), "64 nodes"), (dict(sb=-1), "strides"),
    (dict(sn=-1), "strides"), (dict(d_sb=-1), "strides"), (dict(d_sn=-1), "strides"), (dict(type=1, d=P + 2), "aligned"),
    (dict(scale=0.0), "scale"), (dict(d_scale=-1.0), "scale"), (dict(t=-1.0), "temperature"), (dict(dt=float("nan")), "temperature"),
    (dict(x=None), "null"), (dict(tokens=None), "null"), (dict(u=None), "null"), (dict(choice=None), "null"),
    (dict(accepted=None), "null"), (dict(next=None), "null"), (dict(work=None), "workspace"), (dict(work=P + 4), "workspace")])
def test_verify_refusals(iw, change, what):
    refused(iw, "iw_verify_drafts", VERIFY, change, what)


def test_empty_batches_do_nothing(iw):
    null = dict(q=None, k=None, v=None, out=None)
    assert call(iw, "iw_attention_window", {**WINDOW, **null, "batch": 0})[0] == 0
    assert call(iw, "iw_attention_window", {**WINDOW, **null, "queries": 0})[0] == 0
    assert call(iw, "iw_sample_tokens", {**SAMPLE, "rows": 0, "x": None, "u": None, "work": None})[0] == 0
    assert call(iw, "iw_verify_drafts", {**VERIFY, "batch": 0, "x": None, "u": None, "work": None})[0] == 0


def test_null_structs(iw):
    lib = iw._lib.load()
    for name in FORMS:
        assert getattr(lib, name)(None, None) == -1


def test_struct_images(iw):
    d = iw.drafts
    assert [d._WINDOW_ARGS.format, d._SAMPLE_ARGS.format, d._VERIFY_ARGS.format] == list(FORMS.values())


def test_workspace_sizes(iw):
    value = iw._lib.value
    # 16 bytes for every 256 pieces of 16 bytes, the last perhaps in part
    assert [value("iw_sample_tokens_workspace", 0, 3, n) for n in (1, 4096, 4097, 8192, 8193)] == [48, 48, 96, 96, 144]
    assert value("iw_sample_tokens_workspace", 1, 2, 51865) == 2 * 51 * 16
    assert value("iw_sample_tokens_workspace", 4, 2, 10) == value("iw_sample_tokens_workspace", 0, -1, 10) == -1
    assert value("iw_sample_tokens_workspace", 0, 1, 1 << 23) == -1
    with_draft, without = (value("iw_verify_drafts_workspace", 0, 5, 4, 51865, x) for x in (True, False))
    assert with_draft - without == 5 * 3 * 13 * 16
    assert value("iw_verify_drafts_workspace", 0, 5, 65, 100, True) == -1
    bad = [(-1, 2, 1, 64, 10, 1, 0, 0), (1, 0, 1, 64, 10, 1, 0, 0), (1, 2, -1, 64, 10, 1, 0, 0), (1, 2, 1, 129, 10, 1, 0, 0),
           (1, 2, 1, 64, 0, 1, 0, 0), (1, 2, 1, 64, 10, -1, 0, 0), (1, 2, 1, 64, 10, 1, 1 << 31, 0), (1, 2, 1, 64, 10, 1, 0, -1)]
    assert all(value("iw_attention_window_workspace", *b) == -1 for b in bad)
    assert value("iw_attention_window_workspace", 0, 2, 1, 64, 10, 1, 0, 0) == 0
    # the Python layer asks from 1024 positions on
    for heads, queries, D, cap in ((1, 1, 64, 1023), (4, 8, 128, 1023), (20, 600, 64, 1000)):
        assert value("iw_attention_window_workspace", 1, heads, queries, D, cap, 1 << 30, 0, 0) == 0


def test_python_layer_refuses(iw):
    d = iw.drafts
    z = torch.zeros
    i8 = dict(dtype=torch.int8)
    sc = dict(heads=2, before=3, qk_multiplier=1, qk_shift=1, frac_bits=8, av_multiplier=1, av_shift=1)
    q, k, v = z((1, 2, 128), **i8), z((1, 2, 32, 64), **i8), z((1, 2, 64, 32), **i8)
    for bad, what in (((q, k, v), "GPU tensor"), ((q[0], k, v), "q must be"), ((None, k, v), "q must be"), ((q, k[0], v), "k_cache"),
                      ((q, k, v[..., :16]), "v_cache|GPU"), ((q.float(), k, v), "int8|GPU")):
        with pytest.raises(RuntimeError, match=what):
            d.window_attention(*bad, **sc)
    with pytest.raises(RuntimeError, match="q must be"):
        d.window_attention(q, k, v, **{**sc, "heads": 3})
    x = z((2, 3, 100))
    with pytest.raises(RuntimeError, match="GPU"):
        d.sample_tokens(x, z((2, 3)))
    with pytest.raises(RuntimeError, match="GPU"):
        d.sample_tokens([1.0], z(1))
    with pytest.raises(RuntimeError, match="GPU"):
        d.verify_drafts(x, z((2, 3), dtype=torch.int64), z((2, 2, 100)), z((2, 3)))


def test_draft_decoder_refuses(iw):
    runner = SimpleNamespace(filters=None)
    for kw in (dict(window=-1), dict(sinks=-1), dict(audio=-2), dict(audio_sinks=1 << 31)):
        with pytest.raises(ValueError, match="number of keys"):
            iw.drafts.DraftDecoder(runner, 4, **kw)
    for nodes in (0, 65):
        with pytest.raises(ValueError, match="nodes"):
            iw.drafts.DraftDecoder(runner, nodes)
    with pytest.raises(ValueError, match="filters"):
        iw.drafts.DraftDecoder(SimpleNamespace(filters=iw.LogitFilters(eot=1)), 4)
