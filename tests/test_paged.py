"""Host-side checks of the paged cache's operators and of draft verification, without a GPU: the
wrappers refuse host tensors, and the C ABI answers bad arguments with status codes before any
CUDA call."""
import re
import struct

import pytest
import torch

import gemma_npu_b200 as w8
from gemma_npu_b200 import _lib

BAD, ALIGN, UNSUPPORTED = _lib.W8_ERR_INVALID_ARG, _lib.W8_ERR_ALIGNMENT, _lib.W8_ERR_UNSUPPORTED

# The argument structs of w8a8_b200.h, field by field: pointers (name 0), strides (count) and sizes.
ATTENTION = dict(q=0, k=0, v=0, k_scale=0, v_scale=0, k_tail=0, v_tail=0, k_new=0, v_new=0, out=0, table=0, lens=0, tree=0,
                 depth=0, q_stride=3, k_stride=3, v_stride=3, k_scale_stride=2, v_scale_stride=2, k_tail_stride=3,
                 v_tail_stride=3, k_new_stride=3, v_new_stride=3, out_stride=3, table_stride=1, tree_stride=2,
                 depth_stride=1)
APPEND = dict(k=0, v=0, k_scale=0, v_scale=0, k_tail=0, v_tail=0, table=0, lens=0, k_new=0, v_new=0, path=0, count=0,
              lens_out=0, k_stride=3, v_stride=3, k_scale_stride=2, v_scale_stride=2, k_tail_stride=3, v_tail_stride=3,
              k_new_stride=3, v_new_stride=3, table_stride=1, path_stride=1)
ASSIGN = dict(table=0, lens=0, active=0, free=0, top=0, ok=0, table_stride=1)
VERIFY = dict(logits=0, draft=0, tokens=0, parent=0, uniform=0, path=0, taken=0, token=0, logits_stride=2, draft_stride=2,
              parent_stride=1)
SIZES = {
    "w8_attention_paged": dict(batch=1, heads=4, kv_heads=2, head_dim=64, pages=4, page=16, table_pages=2, n_new=2, window=0,
                               sink=0, dtype=_lib.W8_BF16, scale=1.0),
    "w8_paged_append": dict(batch=1, kv_heads=2, head_dim=64, pages=4, page=16, table_pages=2, n_new=2, steps=2,
                            dtype=_lib.W8_BF16),
    "w8_page_assign": dict(batch=2, table_pages=4, free_pages=8, page=16, room=1, window=0, sink=0),
    "w8_draft_verify": dict(batch=1, n_new=2, vocab=100, dtype=_lib.W8_FP32, temperature=1.0, cap=0.0),
}
FIELDS = {"w8_attention_paged": ATTENTION, "w8_paged_append": APPEND, "w8_page_assign": ASSIGN, "w8_draft_verify": VERIFY}


def args(name, **change):
    """The packed arguments of a small valid-looking call (pointers 4096 apart; optional ones null)."""
    off = {"tree", "depth", "path", "count", "active", "draft", "parent"} if name != "w8_draft_verify" else {"draft", "parent"}
    out, fmt = [], ""
    for i, (field, n) in enumerate(FIELDS[name].items()):
        if n == 0:
            out.append(change.pop(field, 0 if field in off else 4096 * (i + 1)))
            fmt += "Q"
        else:
            value = change.pop(field, 64)
            out += list(value) if isinstance(value, tuple) else [value] * n
            fmt += "%dq" % n
    for field, value in SIZES[name].items():
        value = change.pop(field, value)
        out.append(value)
        fmt += "d" if isinstance(value, float) else "q"
    assert not change
    return struct.pack(fmt, *out)


def run(name, **change):
    lib, a = _lib.lib(), args(name, **change)
    if name == "w8_attention_paged":
        return lib.w8_attention_paged(a, None, 0, None)
    if name == "w8_page_assign":
        return lib.w8_page_assign(a, None, 0, None)
    return getattr(lib, name)(a, None)


@pytest.mark.parametrize("change,status", [
    (dict(heads=5), BAD), (dict(batch=-1), BAD), (dict(window=-1), BAD), (dict(sink=4), BAD), (dict(sink=-1, window=3), BAD),
    (dict(head_dim=96), UNSUPPORTED), (dict(page=48), UNSUPPORTED), (dict(page=8), UNSUPPORTED), (dict(dtype=_lib.W8_FP32), BAD),
    (dict(q=0), BAD), (dict(lens=0), BAD), (dict(k=0), BAD), (dict(k_scale=0), BAD), (dict(table=0), BAD), (dict(k_tail=0), BAD),
    (dict(tree=4096, window=3), BAD), (dict(k_tail=4104), ALIGN), (dict(k=4104), ALIGN), (dict(k_stride=(64, 64, 72)), ALIGN),
    (dict(q_stride=(64, 60, 64)), ALIGN), (dict(k_new_stride=(64, 64, 0)), BAD), (dict(v_stride=(-64, 64, 64)), BAD),
    (dict(scale=0.0), BAD), (dict(scale=float("nan")), BAD), (dict(scale=float("inf")), BAD), (dict(n_new=65537), BAD),
    (dict(table_pages=1 << 27), BAD), (dict(pages=1 << 31), BAD)])
def test_attention_refuses(change, status):
    assert run("w8_attention_paged", **change) == status


@pytest.mark.parametrize("same", ["q", "k", "v", "k_tail", "v_tail", "k_new", "v_new"])
def test_attention_refuses_to_overwrite_an_input(same):
    assert run("w8_attention_paged", out=4096 * (list(ATTENTION).index(same) + 1)) == BAD
    assert b"out must not" in _lib.lib().w8_last_error()


def test_attention_workspace():
    lib = _lib.lib()
    assert lib.w8_attention_paged_workspace_bytes(args("w8_attention_paged")) >= 0
    assert lib.w8_attention_paged_workspace_bytes(args("w8_attention_paged", head_dim=96)) == -1
    assert lib.w8_attention_paged_workspace_bytes(None) == -1


@pytest.mark.parametrize("change,status", [
    (dict(batch=-1), BAD), (dict(head_dim=32), UNSUPPORTED), (dict(page=17), UNSUPPORTED), (dict(dtype=_lib.W8_FP32), BAD),
    (dict(steps=3), BAD), (dict(lens=0), BAD), (dict(lens_out=0), BAD), (dict(k_new=0), BAD), (dict(v=0), BAD),
    (dict(table=0), BAD), (dict(k_tail=4100), ALIGN), (dict(k_stride=(64, 64, 72)), ALIGN),
    (dict(k_new_stride=(64, 64, 60)), ALIGN), (dict(steps=1 << 20, path=4096), BAD)])
def test_append_refuses(change, status):
    assert run("w8_paged_append", **change) == status


def test_append_lens_out_stands_apart():
    """What one CTA writes to lens_out another may yet read from lens, count, path or the table."""
    at = 4096 * (list(APPEND).index("lens_out") + 1)
    for kw in (dict(lens=at), dict(lens=at + 4), dict(lens=at - 12), dict(count=at), dict(count=at - 4), dict(path=at),
               dict(path=at - 4, path_stride=100, steps=2), dict(path=at - 3 * 400 - 4, path_stride=100),
               dict(table=at), dict(table=at - 3 * 400, table_stride=100)):
        assert run("w8_paged_append", batch=4, **kw) == BAD, kw
        assert b"lens_out" in _lib.lib().w8_last_error()


@pytest.mark.parametrize("change,status", [
    (dict(batch=-1), BAD), (dict(batch=8193), BAD), (dict(page=33), UNSUPPORTED), (dict(room=-1), BAD), (dict(window=-1), BAD),
    (dict(sink=2), BAD), (dict(lens=0), BAD), (dict(top=0), BAD), (dict(free=0), BAD), (dict(table=0), BAD), (dict(ok=0), BAD),
    (dict(table_stride=3), BAD), (dict(top=8192), BAD), (dict(lens=4096), BAD), (dict(free=4096 + 8), BAD),
    (dict(batch=8192, table_pages=1 << 17, table_stride=1 << 17, free=0), BAD),
    (dict(batch=100, table_pages=1000, table_stride=1000, free=1 << 30, top=1 << 31, lens=1 << 32), BAD)])
def test_assign_refuses(change, status):
    assert run("w8_page_assign", **change) == status


def test_assign_workspace():
    f = _lib.lib().w8_page_assign_workspace_bytes
    assert f(8, 64) == 0 and f(0, 64) == 0 and f(512, 2048) == 512 * 16


@pytest.mark.parametrize("change,status", [
    (dict(n_new=0), BAD), (dict(n_new=1025), BAD), (dict(vocab=0), BAD), (dict(dtype=3), BAD), (dict(temperature=-1.0), BAD),
    (dict(temperature=1e-4), BAD), (dict(temperature=float("nan")), BAD), (dict(cap=-1.0), BAD), (dict(cap=float("inf")), BAD),
    (dict(logits=0), BAD), (dict(tokens=0), BAD), (dict(uniform=0), BAD), (dict(path=0), BAD), (dict(token=0), BAD)])
def test_verify_refuses(change, status):
    assert run("w8_draft_verify", **change) == status


def test_empty_calls_are_no_ops():
    for name in FIELDS:
        assert run(name, batch=0) == _lib.W8_OK, name
    assert run("w8_attention_paged", n_new=0) == _lib.W8_OK


def test_struct_sizes_match_the_header():
    """8-byte fields, in number as the header declares them."""
    text = re.sub(r"/\*.*?\*/", "", open(_lib.HEADER_PATH).read(), flags=re.S)
    for name in FIELDS:
        body = re.search(r"typedef struct %s_args \{(.*?)\} %s_args;" % (name, name), text, flags=re.S).group(1)
        fields = 0
        for decl in body.split(";"):
            for item in decl.split(","):
                if item.strip():
                    m = re.search(r"\[(\d+)\]", item)
                    fields += int(m.group(1)) if m else 1
        assert len(args(name)) == 8 * fields, name


def test_wrappers_refuse_host_tensors():
    x = torch.zeros((1, 1, 16, 64), dtype=torch.bfloat16)
    p, s = torch.zeros((2, 1, 16, 64), dtype=torch.int8), torch.zeros((2, 1))
    ln, table = torch.zeros(1, dtype=torch.int32), torch.zeros((1, 2), dtype=torch.int32)
    for call in (lambda: w8.attention_paged(x, p, p, s, s, x, x, table, ln, x, x),
                 lambda: w8.paged_append(p, p, s, s, x, x, table, ln, x, x),
                 lambda: w8.page_assign(table, ln, ln, ln, 16), lambda: w8.draft_verify(s[None], ln[None].long(), None)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
