"""The serving step's entry points without a GPU: what they refuse, the struct layouts, and where the tokens of a batch lie, bad pages among them."""
import ctypes as C
import math
import os
import subprocess

import pytest

from gpreempt_amd import capi as gp

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
AT = 1 << 20  # an address that no refused call reads


def test_page_map(tmp_path):
    exe = str(tmp_path / "check")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-fsanitize=address,undefined", "-fno-sanitize-recover", "-I", os.path.join(ROOT, "include"),
                           os.path.join(ROOT, "tests", "page_map_check.cpp"), "-o", exe])
    assert subprocess.run([exe], capture_output=True, text=True).stdout == "ok\n"


def test_struct_layouts(tmp_path):
    """size, and the place of the last member, in C and in the binding"""
    structs = [("gp_kv_cache", gp.KvCache), ("gp_kv_append_params", gp.KvAppendParams), ("gp_paged_attention_params", gp.PagedAttentionParams),
               ("gp_token_logprobs_params", gp.TokenLogprobsParams)]
    members = [(s, n, getattr(m, n).offset) for s, m in structs for n, _ in m._fields_]
    text = "\n".join('_Static_assert(sizeof(%s) == %d, "size");' % (s, C.sizeof(m)) for s, m in structs)
    text += "\n" + "\n".join('_Static_assert(offsetof(%s, %s) == %d, "place");' % m for m in members)
    (tmp_path / "s.c").write_text('#include "gpreempt_hip.h"\n' + text + '\n_Static_assert(GP_E4M3 == %d && GP_ROT_HALVES == %d && GP_ROT_NEIGHBOURS == %d, "values");\n'
                                  % (gp.E4M3, gp.ROT_HALVES, gp.ROT_NEIGHBOURS))
    subprocess.check_call(["gcc", "-fsyntax-only", "-I", os.path.join(ROOT, "include"), str(tmp_path / "s.c")])


def cache(**change):
    c = dict(dtype=gp.F16, kv_heads=2, head_dim=64, page_size=16, pages=10, k=AT, v=AT)
    c.update(change)
    return gp.KvCache(**c)


def append(**change):
    p = dict(dtype=gp.F16, cache=cache(), batch=2, tokens=4, max_new=2, start=AT, kv_len=AT, page_table=AT, table_width=3, heads=4, q=AT, k=AT, v=AT, ld_qkv=512,
             q_out=2 * AT, ld_q_out=256, inv_freq=AT, rot_dim=64, rot_pairs=0)
    p.update(change)
    return gp.KvAppendParams(**p)


def attend(**change):
    p = dict(dtype=gp.F16, cache=cache(), batch=2, tokens=4, max_new=2, max_len=40, start=AT, kv_len=AT, page_table=AT, table_width=3, heads=4, q=AT, ld_q=256, out=2 * AT,
             ld_out=256, scale=0.125, causal=1, work=3 * AT, work_bytes=1 << 40)
    p.update(change)
    return gp.PagedAttentionParams(**p)


def logprobs(**change):
    p = dict(dtype=gp.F32, rows=2, vocab=100, logits=AT, ld=100, tokens=AT, scale=1.0, logprob=AT, entropy=AT, top=3, top_ids=AT, top_logprobs=AT, work=3 * AT, work_bytes=1 << 40)
    p.update(change)
    return gp.TokenLogprobsParams(**p)


def refused(entry, p, says):
    with pytest.raises(gp.GpError) as e:
        gp.launch(entry, p)
    assert e.value.status == gp.OUTOFRANGE and says in str(e.value), str(e.value)
    sizes = {"gp_launch_paged_attention": "gp_paged_attention_work_bytes", "gp_launch_token_logprobs": "gp_token_logprobs_work_bytes"}
    if entry in sizes and says != "workspace":
        assert getattr(gp.lib(), sizes[entry])(C.byref(p), C.byref(C.c_size_t())) == gp.OUTOFRANGE


CACHES = [
    (dict(dtype=gp.BF16), "dtype"), (dict(dtype=gp.F32), "dtype"), (dict(head_dim=96), "head_dim"), (dict(head_dim=0), "head_dim"), (dict(page_size=0), "page_size"),
    (dict(page_size=48), "page_size"), (dict(page_size=256), "page_size"), (dict(kv_heads=0), "shape"), (dict(pages=0), "shape"), (dict(pages=-1), "shape"), (dict(k=None), "keys and values"),
    (dict(v=AT + 8), "aligned"), (dict(dtype=gp.E4M3), "scales"), (dict(dtype=gp.E4M3, k_scale=AT), "scales"),
]


@pytest.mark.parametrize("change,says", CACHES)
def test_caches_that_are_refused(change, says):
    refused("gp_launch_kv_append", append(cache=cache(**change)), says)
    refused("gp_launch_paged_attention", attend(cache=cache(**change)), says)


@pytest.mark.parametrize("change,says", [
    (dict(dtype=gp.F32), "fp16 or bf16"), (dict(dtype=gp.E4M3), "fp16 or bf16"), (dict(batch=0), "positive"), (dict(tokens=0), "positive"), (dict(max_new=0), "positive"),
    (dict(table_width=0), "positive"), (dict(kv_len=None), "null"), (dict(page_table=None), "null"), (dict(k=None), "null"), (dict(v=None), "null"),
    (dict(start=None, tokens=1), "a row for each"), (dict(q_out=None), "place"), (dict(heads=0), "heads"), (dict(ld_qkv=508), "row strides"), (dict(ld_qkv=248), "row strides"),
    (dict(ld_q_out=248), "row strides"), (dict(ld_q_out=-256), "row strides"), (dict(k=AT + 2), "alignment"), (dict(q=AT + 8), "alignment"), (dict(q_out=AT + 4), "alignment"),
    (dict(q_out=AT), "in place"), (dict(rot_dim=24), "rot_dim"), (dict(rot_dim=80), "rot_dim"), (dict(rot_dim=-16), "rot_dim"), (dict(inv_freq=None), "rot_dim"), (dict(rot_pairs=2), "rot_pairs"),
    (dict(batch=1 << 20, max_new=1 << 20, tokens=1 << 30), "too large"),
])
def test_appends_that_are_refused(change, says):
    refused("gp_launch_kv_append", append(**change), says)


@pytest.mark.parametrize("change,says", [
    (dict(dtype=gp.F32), "fp16 or bf16"), (dict(batch=0), "positive"), (dict(tokens=-1), "positive"), (dict(max_new=0), "positive"), (dict(max_len=0), "positive"), (dict(table_width=-3), "positive"),
    (dict(kv_len=None), "null"), (dict(page_table=None), "null"), (dict(q=None), "null"), (dict(out=None), "null"), (dict(start=None, tokens=1), "a row for each"), (dict(heads=3), "multiple"),
    (dict(heads=0), "multiple"), (dict(ld_q=252), "row strides"), (dict(ld_out=248), "row strides"), (dict(q=AT + 2), "alignment"), (dict(out=AT + 8), "alignment"),
    (dict(batch=1 << 16, max_new=1 << 16, tokens=1 << 30), "too large"),
])
def test_attention_that_is_refused(change, says):
    refused("gp_launch_paged_attention", attend(**change), says)


@pytest.mark.parametrize("change,says", [
    (dict(dtype=gp.I32), "dtype"), (dict(dtype=gp.E4M3), "dtype"), (dict(rows=0), "rows"), (dict(rows=1 << 31), "rows"), (dict(vocab=0), "vocab"), (dict(vocab=1 << 30, ld=1 << 30), "vocab"),
    (dict(ld=99), "stride"), (dict(logits=None), "null"), (dict(logits=AT + 2), "aligned"), (dict(top=-1), "alternatives"), (dict(top=33), "alternatives"), (dict(top_ids=None), "place"),
    (dict(top_logprobs=None), "place"), (dict(logprob=None, entropy=None, top=0), "nothing"), (dict(tokens=None), "which tokens"), (dict(scale=-1.0), "scale"), (dict(scale=math.nan), "scale"),
    (dict(scale=math.inf), "scale"),
])
def test_log_probabilities_that_are_refused(change, says):
    refused("gp_launch_token_logprobs", logprobs(**change), says)


def test_workspaces_that_are_refused():
    """what is cut into parts needs one; what is not does without"""
    n = C.c_size_t()
    for entry, size, p in (("gp_launch_paged_attention", "gp_paged_attention_work_bytes", attend(max_len=5000)),
                           ("gp_launch_paged_attention", "gp_paged_attention_work_bytes", attend(max_len=5000, heads=128, cache=cache(kv_heads=64), ld_q=8192, ld_out=8192, max_new=70)),
                           ("gp_launch_token_logprobs", "gp_token_logprobs_work_bytes", logprobs(vocab=200000, ld=200000))):
        gp.check(getattr(gp.lib(), size)(C.byref(p), C.byref(n)))
        assert n.value > 0
        for work, room in ((None, n.value), (AT, n.value - 1), (AT + 8, n.value)):
            p.work, p.work_bytes = work, room
            refused(entry, p, "workspace")
    for size, p in (("gp_paged_attention_work_bytes", attend()), ("gp_token_logprobs_work_bytes", logprobs()), ("gp_token_logprobs_work_bytes", logprobs(rows=1000, vocab=200000, ld=200000))):
        gp.check(getattr(gp.lib(), size)(C.byref(p), C.byref(n)))
        assert n.value == 0


def test_null_params():
    for entry in ("gp_launch_kv_append", "gp_launch_paged_attention", "gp_launch_token_logprobs"):
        assert getattr(gp.lib(), entry)(None, None, None, None) == gp.OUTOFRANGE
    n = C.c_size_t()
    for entry, p in (("gp_paged_attention_work_bytes", attend()), ("gp_token_logprobs_work_bytes", logprobs())):
        assert getattr(gp.lib(), entry)(None, C.byref(n)) == gp.OUTOFRANGE
        assert getattr(gp.lib(), entry)(C.byref(p), None) == gp.OUTOFRANGE
        assert getattr(gp.lib(), entry)(C.byref(p), C.byref(n)) == gp.SUCC
