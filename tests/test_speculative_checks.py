"""Refusals of the drafted-token operators, before any device work: the C entry
points with sizes, alignments and overlaps they do not take, and the Python
layer with tensors that are not what it needs. No GPU."""
import ctypes
import re
import shutil
import struct
import subprocess
from pathlib import Path
from types import SimpleNamespace

import pytest
import torch


def entry(iw, name, args):
    lib = iw._lib.load()
    rc = getattr(lib, name)(*args)
    return rc, lib.iw_last_error().decode()


# any address will do: a refused call reads nothing
P = 1 << 20

PLAN = dict(parents=P, ld=8, counts=None, lengths=None, batch=2, nodes=8, maxp=448, visible=P, positions=P, stream=None)
ATTN = dict(q=P, q_sb=1024, q_st=128, kn=P, kn_sb=1024, kn_st=128, vn=P, vn_sb=1024, vn_st=128, k=P, k_sb=4096,
            k_sh=2048, k_st=64, v=P, v_sb=4096, v_sh=2048, v_sd=4, v_sq=256, lengths=P, visible=P, vis_sb=8,
            counts=None, out=P, o_sb=1024, o_st=128, batch=1, heads=2, nodes=8, D=64, cap=32, qm=3, qs=4, f=8, am=3,
            as_=4, off=16, work=None, stream=None)
ACCEPT = dict(tokens=P, parents=P, choice=P, counts=None, lengths=P, batch=2, nodes=8, eot=-1, path=P, accepted=P,
              next=P, lengths_out=P + 64, layers=1, kn="a", vn="a", kn_sb=1024, kn_st=128, vn_sb=1024, vn_st=128,
              k="a", k_sb=4096, k_sh=2048, k_st=64, v="a", v_sb=4096, v_sh=2048, v_sd=4, v_sq=256, heads=2, D=64,
              cap=32, stream=None)
SCORE = dict(x=P, type=0, rows=2, cols=100, ld=100, scale=1.0, suppress=None, targets=P, logprob=P, entropy=P, top=4,
             ids=P, lps=P, work=None, stream=None)


CACHE_FIELDS = ("layers", "batch", "nodes", "heads", "D", "cap", "kn", "kn_sb", "kn_st", "vn", "vn_sb", "vn_st", "k", "k_sb",
                "k_sh", "k_st", "v", "v_sb", "v_sh", "v_sd", "v_sq")
ACCEPT_ARGS = ("tokens", "parents", "choice", "counts", "lengths", "eot", "path", "accepted", "next", "lengths_out", "stream")


def arguments(name, a):
    """The entry point's arguments; those of the structs as their fields' 64-bit images."""
    def image(values):
        return struct.pack(f"{len(values)}q", *[0 if v is None else v for v in values])
    if name == "iw_attention_tree":
        return image([v for k, v in a.items() if k != "stream"]), None
    if name == "iw_tree_accept":
        arrays = [(ctypes.c_void_p * 1)(P if a[k] == "a" else None) for k in ("kn", "vn", "k", "v")]
        a = dict(a)
        for k, x in zip(("kn", "vn", "k", "v"), arrays):
            a[k] = None if a[k] is None else ctypes.addressof(x)
        KEPT[:] = arrays
        return (image([a[k] for k in CACHE_FIELDS]), *[a[k] for k in ACCEPT_ARGS])
    return tuple(a.values())


KEPT = []  # the arrays that the last image names


def refused(iw, name, args, change, what):
    rc, msg = entry(iw, name, arguments(name, {**args, **change}))
    assert rc == -1 and what in msg, msg


@pytest.mark.parametrize("change,what", [
    (dict(nodes=0), "at most 64 nodes"), (dict(nodes=65, ld=65), "at most 64 nodes"), (dict(ld=7), "tree shape"),
    (dict(batch=-1), "tree shape"), (dict(maxp=0), "max_positions"), (dict(parents=None), "null"),
    (dict(visible=None), "null")])
def test_plan_refusals(iw, change, what):
    refused(iw, "iw_tree_plan", PLAN, change, what)


@pytest.mark.parametrize("change,what", [
    (dict(nodes=0), "1 to 64 nodes"), (dict(nodes=65), "1 to 64 nodes"), (dict(f=0), "frac_bits"),
    (dict(f=14), "frac_bits"), (dict(off=30), "rsqrt_offset"), (dict(D=72), "head_dim"), (dict(D=144), "head_dim"),
    (dict(D=0), "head_dim"), (dict(heads=0), "head_dim"), (dict(cap=0), "cache positions"),
    (dict(cap=1 << 24), "cache positions"), (dict(v_sq=240), "v_sq >= 4"), (dict(v_sd=8), "v_sd == 4"),
    (dict(v_sq=4, v_sd=16), "round_up"), (dict(v_sq=264), "16-byte"), (dict(q=P + 4), "16-byte"),
    (dict(out=P + 8), "16-byte"), (dict(kn_st=130), "16-byte"), (dict(v_sq=4, v_sd=40), "16-byte"),
    (dict(k_st=72), "16-byte"), (dict(q=None), "null"), (dict(lengths=None), "null"), (dict(visible=None), "null"),
    (dict(out=None), "null"), (dict(batch=-1), "attention shape"), (dict(batch=1 << 22), "attention shape"),
    (dict(vis_sb=-1), "attention shape"), (dict(k_st=1 << 25), "2^25"), (dict(kn_st=1 << 25), "2^25"),
    (dict(v_sq=1 << 25), "2^25"), (dict(qm=256), "uint8"), (dict(am=-1), "uint8"), (dict(qs=128), "int8"),
    (dict(as_=-129), "int8"), (dict(off=-1), "rsqrt_offset"), (dict(cap=20000), "workspace"),
    (dict(cap=20000, work=P + 8), "workspace")])
def test_attention_refusals(iw, change, what):
    refused(iw, "iw_attention_tree", ATTN, change, what)


@pytest.mark.parametrize("change,what", [
    (dict(nodes=65), "at most 64 nodes"), (dict(nodes=0), "at most 64 nodes"), (dict(layers=-1), "layers"),
    (dict(lengths_out=P), "lengths_out"), (dict(lengths_out=P + 4), "lengths_out"), (dict(kn=None), "layer pointers"),
    (dict(k="null"), "null tensor"), (dict(vn="null"), "null tensor"), (dict(tokens=None), "null"),
    (dict(next=None), "null"), (dict(kn_st=130), "4-byte"), (dict(k_sh=2050), "4-byte"), (dict(D=20), "head_dim"),
    (dict(cap=0), "cache positions"), (dict(v_sq=4, v_sd=16), "round_up")])
def test_accept_refusals(iw, change, what):
    refused(iw, "iw_tree_accept", ACCEPT, change, what)


@pytest.mark.parametrize("change,what", [
    (dict(type=4), "int8, float32"), (dict(type=-1), "int8, float32"), (dict(rows=-1), "logits shape"),
    (dict(cols=0), "logits shape"), (dict(cols=1 << 23, ld=1 << 23), "logits shape"), (dict(ld=99), "logits shape"),
    (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(scale=1e-40), "scale"),
    (dict(scale=2.0 ** -120), "scale"), (dict(scale=1.2e-38), "scale"), (dict(top=33), "top"), (dict(top=-1), "top"), (dict(cols=3, top=4), "top"),
    (dict(x=None), "null"), (dict(targets=None), "null"), (dict(logprob=None), "null"), (dict(ids=None), "null"),
    (dict(type=1, x=P + 2), "aligned"), (dict(type=2, x=P + 1), "aligned"),
    (dict(cols=100000, ld=100000), "workspace")])
def test_score_refusals(iw, change, what):
    refused(iw, "iw_token_logprobs", SCORE, change, what)


def test_empty_batches_do_nothing(iw):
    for name, args in (("iw_tree_plan", dict(PLAN, batch=0)), ("iw_attention_tree", dict(ATTN, batch=0)),
                       ("iw_token_logprobs", dict(SCORE, rows=0))):
        assert entry(iw, name, arguments(name, args))[0] == 0


def test_null_structs(iw):
    assert entry(iw, "iw_attention_tree", (None, None)) == (-1, "null arguments")
    args = dict(ACCEPT)
    assert entry(iw, "iw_tree_accept", (None, *[args[k] for k in ACCEPT_ARGS])) == (-1, "null arguments")


def test_struct_images(iw):
    """The packed images have the fields of the header's structs, 8 bytes each."""
    text = (Path(__file__).resolve().parents[1] / "include" / "iwhisper_amd.h").read_text()
    for name, image in (("iw_attention_tree_args", iw.speculative._ATTENTION_ARGS), ("iw_tree_caches", iw.speculative._CACHES)):
        body = text[text.index(f"typedef struct {name} {{"):text.index(f"}} {name};")]
        fields = sum(line.count(",") + 1 for line in body.splitlines()[1:] if line.strip().endswith(";"))
        assert image.size == 8 * fields
        assert all(f in ("int64_t", "const") or "*" in line for line in body.splitlines()[1:] for f in line.split()[:1])


def test_workspace_size(iw):
    v = iw._lib.value
    for kind in range(4):
        assert v("iw_token_logprobs_workspace", kind, 8, 51865, 32) >= 0
        assert v("iw_token_logprobs_workspace", kind, 8, 200000, 4) > 0
    for bad in ((0, -1, 5, 0), (0, 1, -5, 0), (0, 1, 5, -1), (4, 1, 5, 0), (-1, 1, 5, 0)):
        assert v("iw_token_logprobs_workspace", *bad) == -1
    for T in (1, 448, 1535):
        assert all(v("iw_attention_tree_workspace", 1, h, 64, D, T) == 0 for h in (1, 40) for D in (64, 128))
    assert 0 < v("iw_attention_tree_workspace", 5, 8, 61, 128, 4096) < 1 << 23
    assert 0 < v("iw_attention_tree_workspace", 1, 1, 1, 16, (1 << 24) - 1) < 1 << 23
    assert v("iw_attention_tree_workspace", 0, 8, 61, 128, 4096) == 0
    for bad in ((-1, 8, 8, 64, 64), (1, 0, 8, 64, 64), (1, 8, 65, 64, 64), (1, 8, 8, 129, 64), (1, 8, 8, 64, 1 << 24)):
        assert v("iw_attention_tree_workspace", *bad) == -1


def i8(*shape):
    return torch.zeros(shape, dtype=torch.int8)


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def i64(*shape):
    return torch.zeros(shape, dtype=torch.int64)


def test_python_layer_refuses(iw):
    sp = iw.speculative
    sc = dict(qk_multiplier=1, qk_shift=1, frac_bits=8, av_multiplier=1, av_shift=1)
    q, k, v = i8(1, 4, 32), i8(1, 2, 8, 16), i8(1, 2, 2, 16, 4)
    with pytest.raises(RuntimeError, match="GPU"):
        sp.tree_attention(q, q, q, k, v, i32(1), i64(1, 4), heads=2, **sc)
    for bad in (None, 3, [1]):
        with pytest.raises(RuntimeError):
            sp.tree_attention(q, bad, q, k, v, i32(1), i64(1, 4), heads=2, **sc)
        with pytest.raises(RuntimeError):
            sp.tree_attention(q, q, q, k, v, bad, i64(1, 4), heads=2, **sc)
    with pytest.raises(RuntimeError, match="whole numbers"):
        sp._pack(sp._CACHES, *[1.5] * 21)
    with pytest.raises(RuntimeError, match="whole numbers"):
        sp._pack(sp._CACHES, *[2 ** 64] * 21)
    with pytest.raises(RuntimeError, match="multiple of heads"):
        sp.tree_attention(q, q, q, k, v, i32(1), i64(1, 4), heads=3, **sc)
    with pytest.raises(RuntimeError, match="1 to 64 nodes"):
        sp.tree_attention(i8(1, 65, 32), q, q, k, v, i32(1), i64(1, 4), heads=2, **sc)
    with pytest.raises(RuntimeError, match="nodes"):
        sp.tree_plan(i32(4))
    with pytest.raises(RuntimeError, match="1 to 64"):
        sp.tree_plan(i32(1, 65))
    with pytest.raises(RuntimeError, match="GPU"):
        sp.tree_plan(i32(1, 8))
    for bad in (0, -1, 2 ** 31, 2 ** 40):
        with pytest.raises(RuntimeError, match="max_positions"):
            sp.tree_plan(i32(1, 8), max_positions=bad)
    with pytest.raises(RuntimeError, match="GPU"):
        sp.token_logprobs(torch.zeros(2, 5))
    with pytest.raises(RuntimeError, match="of each layer"):
        sp.TreeCaches([], [], [], [], heads=2)
    with pytest.raises(RuntimeError, match="of each layer"):
        sp.TreeCaches([q], [q], [k], [], heads=2)
    with pytest.raises(RuntimeError, match="multiple of heads"):
        sp.TreeCaches([q], [q], [k], [v], heads=5)


def test_tree_decoder_refuses(iw):
    with pytest.raises(ValueError, match="filters"):
        iw.speculative.TreeDecoder(SimpleNamespace(filters=iw.LogitFilters(eot=1)), 4)
    for nodes in (0, 65):
        with pytest.raises(ValueError, match="nodes"):
            iw.speculative.TreeDecoder(SimpleNamespace(filters=None), nodes)
    with pytest.raises(ValueError, match="top"):
        iw.speculative.TreeDecoder.step(SimpleNamespace(), i64(1, 4), i32(1, 4), top=0)


def test_kernels_keep_their_values_in_registers(iw, tmp_path):
    """The tree attention's instances spill neither vector nor scalar registers (an early form with
    scalar spills gave wrong probabilities in one lane)."""
    llvm = Path("/opt/rocm/llvm/bin")
    if not (llvm / "llvm-objdump").exists():
        pytest.skip("no llvm-objdump")
    shutil.copy(iw._lib.LIB_PATH, tmp_path / "lib.so")
    subprocess.run([llvm / "llvm-objdump", "--offloading", "lib.so"], cwd=tmp_path, check=True, capture_output=True)
    spills = {}
    for code in sorted(tmp_path.glob("*gfx950*")):
        out = subprocess.run([llvm / "llvm-readelf", "--notes", code], check=True, capture_output=True, text=True).stdout
        for m in re.finditer(r"\.name: +(\S*attn_tree_kernel\S*).*?\.sgpr_spill_count: (\d+).*?\.vgpr_spill_count: (\d+)",
                             out, re.S):
            spills[m[1]] = (int(m[2]), int(m[3]))
    assert len(spills) >= 20 and not any(map(any, spills.values())), spills
