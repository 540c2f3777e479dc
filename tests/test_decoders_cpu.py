"""Products with 4-bit weights, attention behind a shared beginning and over packed prompts, without a GPU: what they refuse, and the struct layouts."""
import ctypes as C
import math
import os
import subprocess

import pytest

from gpreempt_amd import capi as gp
from test_serving_cpu import AT, CACHES, attend, cache

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_struct_layouts(tmp_path):
    structs = [("gp_prefix_attention_params", gp.PrefixAttentionParams), ("gp_packed_attention_params", gp.PackedAttentionParams), ("gp_gemm_w4_params", gp.GemmW4Params)]
    text = "\n".join('_Static_assert(sizeof(%s) == %d, "size");' % (s, C.sizeof(m)) for s, m in structs)
    text += "\n" + "\n".join('_Static_assert(offsetof(%s, %s) == %d, "place");' % (s, n, getattr(m, n).offset) for s, m in structs for n, _ in m._fields_)
    (tmp_path / "s.c").write_text('#include "gpreempt_hip.h"\n' + text)
    subprocess.check_call(["gcc", "-fsyntax-only", "-I", os.path.join(ROOT, "include"), str(tmp_path / "s.c")])


def refused(entry, p, says):
    with pytest.raises(gp.GpError) as e:
        gp.launch(entry, p)
    assert e.value.status == gp.OUTOFRANGE and says in str(e.value), str(e.value)


def w4(**change):
    p = dict(dtype=gp.F16, M=3, N=50, K=256, group=64, A=AT, lda=256, W=AT, ldw=128, scales=AT, ld_scales=4, zeros=AT, ld_zeros=4, C=2 * AT, ldc=50, bias=AT, residual=AT, act=0)
    p.update(change)
    return gp.GemmW4Params(**p)


@pytest.mark.parametrize("change,says", [
    (dict(dtype=gp.F32), "fp16 or bf16"), (dict(dtype=gp.E4M3), "fp16 or bf16"), (dict(M=0), "positive"), (dict(N=-1), "positive"), (dict(K=0), "positive"), (dict(M=(1 << 30) + 1), "2^30"), (dict(N=(1 << 30) + 1, ldc=1 << 31), "2^30"), (dict(K=(1 << 30) + 64, lda=1 << 31, ldw=1 << 30, ld_scales=1 << 30, ld_zeros=1 << 30), "2^30"), (dict(group=0), "group"),
    (dict(group=16), "group"), (dict(group=256), "group"), (dict(K=224, lda=224), "multiple of the group"), (dict(lda=248), "lda"), (dict(lda=260), "lda"), (dict(ldw=120), "ldw"), (dict(ldw=112), "ldw"),
    (dict(ld_scales=3), "row strides"), (dict(ld_zeros=3), "row strides"), (dict(ldc=49), "ldc"), (dict(A=None), "null"), (dict(W=None), "null"), (dict(scales=None), "null"), (dict(C=None), "null"),
    (dict(A=AT + 8), "16-byte"), (dict(W=AT + 4), "16-byte"), (dict(C=2 * AT + 1), "elements"), (dict(scales=AT + 1), "elements"), (dict(bias=AT + 1), "elements"), (dict(residual=AT + 1), "elements"),
    (dict(act=3), "act"), (dict(act=-1), "act"), (dict(lda=-256), "lda"), (dict(ldc=-50), "ldc"),
])
def test_products_that_are_refused(change, says):
    refused("gp_launch_gemm_w4", w4(**change), says)


def prefix(shared_len=32, shared_table=AT, variant=0, **change):
    return gp.PrefixAttentionParams(attention=attend(**change), shared_len=shared_len, shared_table=shared_table, variant=variant)


def refused_prefix(p, says):
    refused("gp_launch_prefix_attention", p, says)
    if says != "workspace":
        assert gp.lib().gp_prefix_attention_work_bytes(C.byref(p), C.byref(C.c_size_t())) == gp.OUTOFRANGE


@pytest.mark.parametrize("change,says", CACHES)
def test_caches_that_are_refused(change, says):
    refused_prefix(prefix(cache=cache(**change)), says)


@pytest.mark.parametrize("change,says", [
    (dict(shared_len=-16), "whole pages"), (dict(shared_len=24), "whole pages"), (dict(shared_table=None), "shared pages"), (dict(dtype=gp.F32), "fp16 or bf16"), (dict(batch=0), "positive"),
    (dict(max_new=0), "positive"), (dict(max_len=0), "positive"), (dict(kv_len=None), "null"), (dict(q=None), "null"), (dict(out=None), "null"), (dict(start=None, tokens=1), "a row for each"),
    (dict(heads=3), "multiple"), (dict(ld_q=252), "row strides"), (dict(ld_out=248), "row strides"), (dict(q=AT + 2), "alignment"), (dict(out=AT + 8), "alignment"), (dict(scale=math.nan), "scale"),
    (dict(scale=2.0 ** -110), "scale"), (dict(scale=math.inf), "scale"), (dict(variant=3), "variant"), (dict(variant=-1), "variant"), (dict(shared_len=1 << 30 | 16), "2^30"),
    (dict(shared_len=0, variant=gp.PREFIX_TOGETHER), "together"), (dict(max_new=40, variant=gp.PREFIX_TOGETHER), "together"), (dict(batch=10000, tokens=20000, variant=gp.PREFIX_TOGETHER), "together"),
])
def test_shared_beginnings_that_are_refused(change, says):
    refused_prefix(prefix(**change), says)


def test_a_workspace_that_is_refused():
    n, p = C.c_size_t(), prefix(variant=gp.PREFIX_TOGETHER)
    gp.check(gp.lib().gp_prefix_attention_work_bytes(C.byref(p), C.byref(n)))
    assert n.value > 0
    for work, room in ((None, n.value), (AT, n.value - 1), (AT + 8, n.value)):
        p.attention.work, p.attention.work_bytes = work, room
        refused_prefix(p, "workspace")


def packed(**change):
    p = dict(dtype=gp.F16, batch=2, tokens=100, max_len=60, start=AT, heads=4, kv_heads=2, head_dim=64, q=AT, ld_q=512, k=AT + 512, v=AT + 768, ld_kv=512, out=2 * AT, ld_out=256, scale=0.125, causal=1)
    p.update(change)
    return gp.PackedAttentionParams(**p)


@pytest.mark.parametrize("change,says", [
    (dict(dtype=gp.F32), "fp16 or bf16"), (dict(dtype=gp.E4M3), "fp16 or bf16"), (dict(batch=0), "positive"), (dict(tokens=0), "positive"), (dict(max_len=0), "positive"), (dict(max_len=-5), "positive"),
    (dict(start=None), "null"), (dict(q=None), "null"), (dict(k=None), "null"), (dict(v=None), "null"), (dict(out=None), "null"), (dict(heads=3), "multiple"), (dict(heads=0), "multiple"),
    (dict(kv_heads=0), "multiple"), (dict(head_dim=96), "head_dim"), (dict(head_dim=256), "head_dim"), (dict(ld_q=252), "row strides"), (dict(ld_q=248), "row strides"), (dict(ld_kv=120), "row strides"),
    (dict(ld_out=248), "row strides"), (dict(ld_out=-256), "row strides"), (dict(ld_kv=(1 << 25) + 8), "2^25"), (dict(q=AT + 8), "alignment"), (dict(k=AT + 2), "alignment"), (dict(v=AT + 8), "alignment"), (dict(out=2 * AT + 8), "alignment"),
    (dict(scale=math.nan), "scale"), (dict(scale=2.0 ** 101), "scale"), (dict(tokens=1 << 30, max_len=1 << 30), "too large"),
    (dict(tokens=1 << 29, max_len=1 << 28, batch=1 << 20), "too large"),
])
def test_packed_prompts_that_are_refused(change, says):
    refused("gp_launch_packed_attention", packed(**change), says)


def test_null_params():
    for entry in ("gp_launch_gemm_w4", "gp_launch_prefix_attention", "gp_launch_packed_attention"):
        assert getattr(gp.lib(), entry)(None, None, None, None) == gp.OUTOFRANGE
    n = C.c_size_t()
    assert gp.lib().gp_prefix_attention_work_bytes(None, C.byref(n)) == gp.OUTOFRANGE
    assert gp.lib().gp_prefix_attention_work_bytes(C.byref(prefix()), None) == gp.OUTOFRANGE
    assert gp.lib().gp_prefix_attention_work_bytes(C.byref(prefix()), C.byref(n)) == gp.SUCC


def test_counters_in_front_of_a_workspace(tmp_path):
    exe = str(tmp_path / "check")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-I", os.path.join(ROOT, "include"), os.path.join(ROOT, "tests", "join_counters_check.cpp"), "-o", exe])
    assert subprocess.run([exe], capture_output=True, text=True).stdout == "ok\n"


def work_bytes(variant, batch, shared, own, heads, kv_heads, dim, dtype):
    c = cache(dtype=dtype, kv_heads=kv_heads, head_dim=dim, page_size=64, pages=1 << 20, **(dict(k_scale=AT, v_scale=AT) if dtype == gp.E4M3 else {}))
    p = prefix(shared, cache=c, dtype=gp.F16, batch=batch, tokens=batch, max_new=1, start=None, max_len=shared + own, table_width=-(-(shared + own) // 64), heads=heads, ld_q=heads * dim, ld_out=heads * dim,
               variant=variant)
    n = C.c_size_t()
    gp.check(gp.lib().gp_prefix_attention_work_bytes(C.byref(p), C.byref(n)))
    return n.value


@pytest.mark.parametrize("shared", [8192, 16384, 32768])
def test_one_sequence_more_does_not_change_how_the_shared_keys_are_cut(shared):
    """about as many sequences as fill the chip once: the workspace, of which a part of the shared keys takes 66 KB, grows by a sequence's share of it"""
    sizes = [work_bytes(gp.PREFIX_TOGETHER, batch, shared, 100, 32, 8, 128, gp.E4M3) for batch in (62, 63, 64)]
    assert max(sizes) - min(sizes) < 1 << 20, sizes


@pytest.mark.parametrize("heads, kv_heads, dim, dtype, shared, each, together", [
    (32, 8, 128, gp.E4M3, 1024, 48, 96), (32, 8, 128, gp.E4M3, 4096, 16, 48), (32, 8, 128, gp.E4M3, 16384, 8, 12), (32, 8, 128, gp.F16, 1024, 32, 64), (32, 8, 128, gp.F16, 16384, 4, 6),
    (8, 1, 128, gp.E4M3, 8192, 48, 128), (32, 2, 128, gp.F16, 4096, 32, 96), (12, 12, 64, gp.F16, 1024, 12, 32), (12, 12, 64, gp.F16, 4096, 6, 12),
])
def test_the_launcher_chooses_what_is_faster(heads, kv_heads, dim, dtype, shared, each, together):
    """numbers of sequences on either side of where measurements cross"""
    for batch, variant in ((each, gp.PREFIX_EACH), (together, gp.PREFIX_TOGETHER)):
        sizes = {v: work_bytes(v, batch, shared, 100, heads, kv_heads, dim, dtype) for v in (gp.PREFIX_AUTO, gp.PREFIX_EACH, gp.PREFIX_TOGETHER)}
        assert sizes[gp.PREFIX_EACH] != sizes[gp.PREFIX_TOGETHER]
        assert sizes[gp.PREFIX_AUTO] == sizes[variant], (batch, sizes)


def test_the_shared_tiles_leave_a_place_for_whoever_reads_the_flag():
    """behind 131072 tokens two workgroups to each of 256 compute units, less one for each XCD: 63 parts of eight heads, of 66 KB each"""
    part, rows = (128 // 2 + 2) * 256 * 4, 16 * (128 + 2) * 4  # bytes of what 128 rows, and 16, come to
    others = 69632 + 8 * 5 * rows + 8 * 32 * 2 * rows  # counters, own keys, parts of a sequence that ends within what is shared
    assert (work_bytes(gp.PREFIX_TOGETHER, 5, 131072, 100, 32, 8, 128, gp.F16) - others) // part == 8 * 63
