"""Host-side checks of the decoding operators, without a GPU: the wrappers refuse host
tensors, and the C ABI answers bad arguments with status codes before any CUDA call."""
import struct

import pytest
import torch

import gemma_npu_b200 as w8
from gemma_npu_b200 import _lib

# The argument structs of w8a8_b200.h: pointers, then 64-bit integers (and a double).
TREE_ARGS = struct.Struct("12Q33qd")
APPEND_ARGS = struct.Struct("11Q25q")
EVICT_ARGS = struct.Struct("8Q21q")


def tree_args(**change):
    """The packed arguments of a small valid-looking attention_tree call (pointers 256 apart)."""
    p = {name: 4096 + 256 * i for i, name in enumerate(
        ["q", "k", "v", "k_new", "v_new", "out", "lens", "tree", "depth", "weights", "weights_out", "draft_weights"])}
    p.update(tree=0, depth=0, weights=0, weights_out=0, draft_weights=0)
    s = {name: (64, 64, 64) for name in ["qs", "ks", "vs", "kns", "vns", "os"]}
    n = dict(B=1, H=4, KV=2, D=64, S=16, N=2, window=0, dtype=_lib.W8_BF16, scale=1.0)
    for name, v in change.items():
        next(d for d in (p, s, n) if name in d)[name] = v
    return TREE_ARGS.pack(*p.values(), *(x for v in s.values() for x in v), 4, 2, 0, 0, 0, 0, 0, *n.values())


@pytest.mark.parametrize("change,status", [
    (dict(H=5), _lib.W8_ERR_INVALID_ARG), (dict(B=-1), _lib.W8_ERR_INVALID_ARG), (dict(window=-1), _lib.W8_ERR_INVALID_ARG),
    (dict(D=96), _lib.W8_ERR_UNSUPPORTED), (dict(dtype=_lib.W8_FP32), _lib.W8_ERR_INVALID_ARG), (dict(q=0), _lib.W8_ERR_INVALID_ARG),
    (dict(lens=0), _lib.W8_ERR_INVALID_ARG), (dict(k=0), _lib.W8_ERR_INVALID_ARG), (dict(tree=4096, window=3), _lib.W8_ERR_INVALID_ARG),
    (dict(weights=4096), _lib.W8_ERR_INVALID_ARG), (dict(k=4104), _lib.W8_ERR_ALIGNMENT), (dict(ks=(64, 64, 60)), _lib.W8_ERR_ALIGNMENT),
    (dict(scale=0.0), _lib.W8_ERR_INVALID_ARG), (dict(scale=float("nan")), _lib.W8_ERR_INVALID_ARG),
    (dict(N=65537), _lib.W8_ERR_INVALID_ARG)])
def test_attention_tree_refuses(change, status):
    assert _lib.lib().w8_attention_tree(tree_args(**change), None, 0, None) == status


@pytest.mark.parametrize("same", ["q", "k", "v", "k_new", "v_new"])
def test_attention_tree_refuses_to_overwrite_an_input(same):
    at = {name: 4096 + 256 * i for i, name in enumerate(["q", "k", "v", "k_new", "v_new"])}[same]
    assert _lib.lib().w8_attention_tree(tree_args(out=at), None, 0, None) == _lib.W8_ERR_INVALID_ARG
    assert b"out must not" in _lib.lib().w8_last_error()


def test_in_place_needs_one_layout():
    """Weights updated in place through strides other than their own would mix up the heads."""
    raw = bytearray(tree_args(B=2, weights=4096, weights_out=4096, draft_weights=8192))
    strides = 12 * 8 + (18 + 3) * 8  # weights_stride[2], weights_out_stride[2]
    raw[strides:strides + 32] = struct.pack("4q", 32, 16, 16, 32)
    assert _lib.lib().w8_attention_tree(bytes(raw), None, 0, None) == _lib.W8_ERR_INVALID_ARG
    assert b"other strides" in _lib.lib().w8_last_error()
    for w_to, p_to in ((16384, 24576), (16384, 40960), (32768, 24576)):
        evict = EVICT_ARGS.pack(4096, 8192, 16384, 24576, 4096, w_to, p_to, 8192, *[128] * 6, 32, 16, 32, 16, 16, 32, 16, 32,
                                2, 2, 16, 128, 4, 0, 0)
        assert _lib.lib().w8_cache_evict(evict, 4096, 1 << 20, None) == _lib.W8_ERR_INVALID_ARG
        assert b"other strides" in _lib.lib().w8_last_error()


def test_empty_attention_is_a_no_op():
    assert _lib.lib().w8_attention_tree(tree_args(B=0), None, 0, None) == _lib.W8_OK
    assert _lib.lib().w8_attention_tree(tree_args(N=0), None, 0, None) == _lib.W8_OK


def test_struct_sizes_match_the_header():
    """8-byte fields, in number as the header declares them."""
    import re

    text = re.sub(r"/\*.*?\*/", "", open(_lib.HEADER_PATH).read(), flags=re.S)
    for name, packed in (("w8_attention_tree_args", TREE_ARGS), ("w8_cache_append_args", APPEND_ARGS),
                         ("w8_cache_evict_args", EVICT_ARGS)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, flags=re.S).group(1)
        fields = 0
        for decl in body.split(";"):
            for item in decl.split(","):
                if item.strip():
                    m = re.search(r"\[(\d+)\]", item)
                    fields += int(m.group(1)) if m else 1
        assert packed.size == 8 * fields, name


def test_cluster_barriers_find_their_warps_converged():
    """`barrier.cluster.*.aligned` needs every thread of the warp at it: the one place that issues it
    converges the warp first."""
    import glob
    import os

    csrc = os.path.join(os.path.dirname(_lib.__file__), "csrc")
    for path in glob.glob(os.path.join(csrc, "*.cu*")):
        text = open(path).read()
        if os.path.basename(path) == "common.cuh":
            body = text.split("void cluster_sync() {", 1)[1].split("}", 1)[0]
            assert body.index("__syncwarp();") < body.index("barrier.cluster.arrive")
            text = text.replace(body, "")
        assert "barrier.cluster." not in text, path


def test_lens_out_stands_apart():
    """What one CTA writes to lens_out another may yet read from lens, seen or path: the same array, or
    one that overlaps it at another address, is refused."""
    def append(lens=4096, path=0, seen=16384, lens_out=32768, positions=24576, stride=3, draft=0):
        return APPEND_ARGS.pack(4096, 8192, 12288, 16384, lens, path, 0, draft, positions, seen, lens_out, *[128] * 12,
                                stride, 0, 0, 0, 0, 64, 16, 4, 2, 64, 8, 8, 128)

    run = _lib.lib().w8_cache_append
    for kw in (dict(lens=32768), dict(lens=32768 + 4), dict(lens=32768 - 12), dict(seen=32768), dict(seen=32768 + 12),
               dict(seen=32768 - 4), dict(path=32768, stride=8), dict(path=32768 - 4, stride=8), dict(path=32768 - 3 * 32 - 28, stride=8)):
        assert run(append(**kw), None) == _lib.W8_ERR_INVALID_ARG, kw
        assert b"lens_out" in _lib.lib().w8_last_error()
    # Beside it, between the rows of a path, and positions that are not kept: nothing of that to refuse
    # (and so that nothing runs, draft weights without weights, which is looked at next).
    for kw in (dict(lens=32768 + 16), dict(seen=32768 - 16), dict(path=32768 - 32, stride=100), dict(seen=32768, positions=0)):
        assert run(append(draft=4096, **kw), None) == _lib.W8_ERR_INVALID_ARG
        assert b"draft_weights need weights" in _lib.lib().w8_last_error(), kw

    def evict(lens):
        return EVICT_ARGS.pack(4096, 4096, 4096, 4096, lens, 4096, 4096, 8192, *[128] * 6, *[16] * 8, 4, 1, 16, 128, 4, 0, 0)

    for lens in (8192, 8188, 8204):
        assert _lib.lib().w8_cache_evict(evict(lens), 4096, 1 << 20, None) == _lib.W8_ERR_INVALID_ARG
        assert b"lens_out" in _lib.lib().w8_last_error()


def test_evict_refuses():
    def args(budget=4, sink=0, recent=0, lens=4096, lens_out=8192, row=128):
        return EVICT_ARGS.pack(4096, 4096, 4096, 4096, lens, 4096, 4096, lens_out, *[128] * 6, *[16] * 8, 1, 1, 16, row,
                               budget, sink, recent)

    run = _lib.lib().w8_cache_evict
    for a in (args(budget=0), args(sink=-1), args(sink=2, recent=3), args(lens=0), args(lens_out=4096)):
        assert run(a, 4096, 1 << 20, None) == _lib.W8_ERR_INVALID_ARG
    assert run(args(row=24), 4096, 1 << 20, None) == _lib.W8_ERR_ALIGNMENT
    assert run(args(), 4096, 8, None) == _lib.W8_ERR_INVALID_ARG
    assert b"workspace" in _lib.lib().w8_last_error()


def test_select_refuses():
    def run(beams=2, vocab=10, n=2, pad=0, dtype=_lib.W8_FP32, slot=0, logits=4096):
        return _lib.lib().w8_beam_select(logits, dtype, vocab * beams, vocab, 4096, None, pad, 0.0, 1, beams, vocab, n, slot,
                                         4096, 4096, 4096, 4096, 1 << 20, None)

    for kw in (dict(n=21), dict(n=0), dict(pad=10), dict(pad=-1), dict(dtype=3), dict(slot=1, n=3), dict(logits=None)):
        assert run(**kw) == _lib.W8_ERR_INVALID_ARG, kw
    assert run(beams=33) == _lib.W8_ERR_UNSUPPORTED and run(n=65, vocab=100) == _lib.W8_ERR_UNSUPPORTED
    assert run(logits=4098) == _lib.W8_ERR_ALIGNMENT


@pytest.mark.parametrize("cap", [float("nan"), float("inf"), 1e-31, 1e31])
def test_select_refuses_caps_it_cannot_scale(cap):
    assert _lib.lib().w8_beam_select(4096, _lib.W8_FP32, 20, 10, 4096, None, 0, cap, 1, 2, 10, 2, 0, 4096, 4096, 4096, 4096,
                                     1 << 20, None) == _lib.W8_ERR_INVALID_ARG
    assert b"cap must be" in _lib.lib().w8_last_error()


def test_binding_loads_a_library_under_any_name(tmp_path):
    """The library's path need not be UTF-8 (a process of its own: this one's binding stays bound)."""
    import os
    import shutil
    import subprocess
    import sys

    from gemma_npu_b200 import decode

    try:
        odd = os.path.join(os.fsencode(str(tmp_path)), b"lib-\xff.so")
        os.symlink(os.fsencode(_lib.LIB_PATH), odd)
    except OSError:
        shutil.copy(_lib.LIB_PATH, tmp_path / "lib.so")
        odd = os.fsencode(str(tmp_path / "lib.so"))
    code = ("import importlib.util, os, sys, torch\n"
            "spec = importlib.util.spec_from_file_location('_decode', sys.argv[1])\n"
            "m = importlib.util.module_from_spec(spec); spec.loader.exec_module(m)\n"
            "m.bind(sys.argv[2], print)\n"
            "try:\n    m.bind(sys.argv[2] + '.none', print)\n"
            "except ValueError as e:\n    assert str(e).startswith('cannot load')\n"
            "else:\n    raise SystemExit(1)\n")
    subprocess.run([sys.executable, "-c", code, decode.BINDING_PATH, odd], check=True, timeout=300)


def test_wrappers_refuse_host_tensors():
    x = torch.zeros((1, 1, 4, 64), dtype=torch.bfloat16)
    ln = torch.zeros(1, dtype=torch.int32)
    w = torch.zeros((1, 1, 4))
    for call in (lambda: w8.attention_tree(x, x, x, ln, x, x), lambda: w8.cache_append(x, x, x, x, ln),
                 lambda: w8.cache_evict(x, x, w, w.int(), ln, 2), lambda: w8.beam_select(w, w[0]),
                 lambda: w8.cache_reorder(x, torch.zeros((1, 1), dtype=torch.int64))):
        with pytest.raises(ValueError, match="CUDA"):
            call()
