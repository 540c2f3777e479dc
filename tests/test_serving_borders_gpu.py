"""The serving step's kernels at the borders of what they take: scales, NaN, probabilities and lengths (definitions and callers: serving.py, test_serving_gpu.py)."""
import pytest
import torch

import serving as S
import test_serving_gpu as T

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", ["bf16"])
def test_append_to_a_page_whose_scale_attention_takes_as_a_border(gp, dt):
    """8 bits: what append keeps, rescales and writes reads back on the scale that attention takes, 2^-60 .. 2^60, whatever scale the page came with or its values ask for"""
    lens, page, dim = [5, 5, 5, 5, 1, 5], 16, 64
    seqs = S.Sequences(lens, None, page, T.gen(1))
    sizes = [0.0, 2.0 ** -64, 2.0 ** 62, 1.0, 2.0 ** 75, 2.0 ** 60]  # of the new tokens
    before = [2.0 ** -130, 2.0 ** -70, 2.0 ** 70, 2.0 ** -126, 1.0, float("inf")]  # the scales of their pages (the fifth begins)

    def change(a):
        for b, size in enumerate(sizes):
            a.qkv[b] = (a.qkv[b].double().clamp(-2, 2) * size).to(S.TORCH[dt])
            for n in ("k_scale", "v_scale"):
                a.cache[n][int(seqs.table[b, 0])] = before[b]

    a = T.Append(gp, dt, "e4m3", seqs, 2, 2, dim, 0, "halves", 2, change=change)
    a.launch()
    left = a.left()
    for name, first in (("k", 2), ("v", 4)):
        new = a.part(first, 2).double()
        for b, n in enumerate(lens):
            at = int(seqs.table[b, 0])
            scale = left[name + "_scale"][at].double().clamp(2.0 ** -60, 2.0 ** 60)[:, None]
            got = left[name][at].double() * scale[..., None]  # heads x slots x dim
            most = 448 * scale
            want = torch.maximum(torch.minimum(new[b], most), -most)
            step = torch.maximum(2.0 ** -4 * want.abs(), 2.0 ** -10 * scale)  # half a step of e4m3, of its smallest values
            assert ((got[:, n - 1] - want).abs() <= step).all(), (name, b)
            old = a.cache[name][at].double() * min(max(before[b], 2.0 ** -60), 2.0 ** 60)
            for slot in range(n - 1):
                step = torch.maximum(2.0 ** -4 * old[:, slot].abs(), 2.0 ** -10 * scale)
                assert ((got[:, slot] - old[:, slot]).abs() <= step).all(), (name, b, slot)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [40, 9001, 70000])
def test_alternatives_next_to_a_nan_of_either_kind(gp, dt, vocab):
    """a signalling or a quiet NaN right behind the row's largest logit, whose neighbours are all small: the alternatives are the others, in order"""
    ints, bad = {"f32": (torch.int32, (0x7F800001, 0x7FC00000)), "f16": (torch.int16, (0x7C01, 0x7E00)), "bf16": (torch.int16, (0x7F81, 0x7FC0))}[dt]
    rng = T.gen(3)
    x = torch.randn((4, vocab), generator=rng)
    vec = 4 if dt == "f32" else 8
    for at in range(0, vocab, 512 * vec):  # what eight threads next to each other read
        x[:, at: at + 8 * vec] = -50.0 - torch.arange(vocab)[at: at + 8 * vec] / 4096
    x = x.to(S.TORCH[dt])
    x[:, 0] = 9.0
    for r in range(4):
        x.view(ints)[r, 2 + r // 2] = bad[r % 2]
    a = T.Logprobs(gp, dt, x, torch.tensor([0, 1, 2, 3]), 20)
    assert torch.equal(a.room.cpu().view(ints), x.view(ints).flatten())  # (no copy has made them quiet)
    a.launch()
    got = a.left()
    assert torch.equal(got["ids"], S.logprobs(x, torch.zeros(4), 1.0, 20)[2])
    assert got["logprob"].isnan().all() and got["entropy"].isnan().all() and got["values"].isnan().all()


@pytest.mark.parametrize("cache", ["same", "e4m3"])
@pytest.mark.parametrize("dt", T.DTS)
@pytest.mark.parametrize("lens, news, heads, kv_heads, dim", [([3000, 700], None, 8, 2, 128), ([2000, 1500, 1000, 300], [70, 66, 67, 80], 16, 16, 64)])
def test_attention_to_many_unlikely_keys(gp, dt, cache, lens, news, heads, kv_heads, dim):
    """One key takes nearly everything and its values are zero: the result is what the others, each 2^26 times less likely, add up to."""
    seqs = S.Sequences(lens, news, 64, T.gen(4))
    a = T.Attend(gp, dt, dt if cache == "same" else cache, seqs, heads, kv_heads, dim, False, 5, scale=1.0)
    a.q[:] = 0.0
    a.q[:, ::dim] = 18.0  # e^18 = 2^26
    if cache == "e4m3":
        for n in ("k_scale", "v_scale"):
            a.cache[n][:] = 1.0
    one, zero = (torch.tensor(x).to(a.cache["k"].dtype) for x in (1.0, 0.0))
    a.cache["k"][:], a.cache["v"][:] = zero, one
    for b in range(seqs.batch):
        page, slot = seqs.place(b, b)
        a.cache["k"][page, :, slot, 0], a.cache["v"][page, :, slot] = one, zero
    for n, x in a.cache.items():
        a.dev[n].copy_(x)
    a.dev["q"].copy_(a.q)
    a.launch()
    a.check()


@pytest.mark.parametrize("scale", [2.0 ** -100, 2.0 ** 100])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_logprobs_at_the_borders_of_the_scale(gp, dt, scale):
    """all tokens are alike, the type's lowest value among them; one takes everything"""
    x = torch.randn((3, 40000), generator=T.gen(6)).to(S.TORCH[dt])
    x[:, 7], x[1, 9] = 100.0, -torch.inf
    if scale < 1:
        x[2, 11] = torch.finfo(S.TORCH[dt]).min
    a = T.Logprobs(gp, dt, x, torch.tensor([7, 8, 11]), 5, scale)
    a.launch()
    a.check()


# ---- many query rows of 128 values -------------------------------------------------------------------------------------------


@pytest.mark.parametrize("cache", ["same", "e4m3"])
@pytest.mark.parametrize("dt", T.DTS)
@pytest.mark.parametrize("page", [16, 64])
def test_many_rows_of_128_values_in_parts(gp, dt, cache, page):
    """blocks whose keys are cut into two parts, and one of a single part"""
    seqs = S.Sequences([1300, 1100, 900, 70], [70, 66, 80, 70], page, T.gen(10), tail=1)
    a = T.Attend(gp, dt, dt if cache == "same" else cache, seqs, 16, 16, 128, True, 11)
    info = a.launch()
    assert tuple(info.shape)[:2] == (2, 64)
    a.check()
    first = a.left()
    a.launch()
    assert torch.equal(a.left(), first)


@pytest.mark.parametrize("cache", ["same", "e4m3"])
@pytest.mark.parametrize("dt", T.DTS)
def test_many_rows_of_128_values_over_more_keys_than_a_window_of_pages(gp, dt, cache):
    """one part of 22 tiles of keys, whose pages and scales are looked up sixteen at a time; pages that are not there in either window"""
    seqs = S.Sequences([1400, 70], [67, 66], 64, T.gen(12), holes={(0, 3): -1, (0, 17): 10 ** 6})
    a = T.Attend(gp, dt, dt if cache == "same" else cache, seqs, 130, 130, 128, True, 13)
    info = a.launch()
    assert tuple(info.shape)[:2] == (1, 260)
    a.check()


def test_many_rows_are_taken_in_blocks_of_128(gp):
    """the cases of test_serving_gpu.py reach the kernel that they are about"""
    shapes = []
    for lens, news, page, heads, kv_heads, dim, causal in T.MANY:
        seqs = S.Sequences(lens, news, page, T.gen(14), tail=1)
        shapes.append(tuple(T.Attend(gp, "f16", "f16", seqs, heads, kv_heads, dim, causal, 15).launch().shape)[:2])
    assert shapes == [(2, 64), (4, 64), (4, 64), (1, 64)]  # (blocks times parts, heads times sequences; the third: 390 rows, and 3 * 2 * 2 tiles are more than 700 keys)


# ---- stopped with results that wait for the others' ------------------------------------------------------------------------------


def joined_calls(gp):
    """calls whose results are joined from parts, of more tiles than there are claim counters"""
    rng = T.gen(20)
    yield T.Attend(gp, "f16", "f16", S.Sequences([2000, 700, 1], None, 64, rng), 8, 4, 64, True, 21)
    yield T.Attend(gp, "bf16", "e4m3", S.Sequences([1500, 300, 900], [6, 1, 8], 32, rng), 16, 4, 128, True, 22)
    yield T.Attend(gp, "bf16", "e4m3", S.Sequences([1300, 1100, 900, 70], [70, 66, 80, 70], 64, rng), 16, 16, 128, True, 23)
    yield T.Attend(gp, "f16", "f16", S.Sequences([1300, 1100, 900, 70], [70, 66, 80, 70], 16, rng), 16, 16, 128, True, 24)
    yield T.Logprobs(gp, "bf16", torch.randn((40, 70000), generator=rng).bfloat16(), torch.arange(40), 20)


@pytest.mark.parametrize("which", range(5))
def test_stopped_between_the_parts_of_a_result(gp, which):
    """32 claim counters, served by a workgroup each: the first tile raises the flag, which its workgroup sees in front of its next one; the first result's other parts have
    not been made then"""
    call = list(joined_calls(gp))[which]
    assert call.p.work_bytes and call.launch().total_tiles > 32
    want = call.left()
    T.clean(call)
    flag = gp.Flag()
    st = gp.BlpState(1, flag, 32)
    call.launch(st.ctx(inject_at=0, max_workgroups=1, poll_every=1))
    call.left()
    counters = call.work[:1024].view(torch.int32)
    assert flag.get() == 1 and st.stop_index() == 0 and int(counters[0]) > 0 and not T.same(call.left(), want)
    flag.set(0)
    st.clear_stop()
    call.launch(st.ctx(max_workgroups=1, poll_every=1))
    assert T.same(call.left(), want) and not counters.any()


# ---- an append of so many tiles that a claim stands for several -------------------------------------------------------------------


@pytest.mark.parametrize("cache", ["f16", "e4m3"])
def test_append_of_several_tiles_a_claim(gp, cache):
    """64 sequences of a few new tokens each under a bound of 3000: most tiles find nothing to do, and those that do share a claim with others; as one launch, and stopped and resumed"""
    news = [1 + i * 7 % 23 for i in range(64)]
    seqs = S.Sequences([n + i * 11 % 40 for i, n in enumerate(news)], news, 16, T.gen(30), max_new=3000, tail=1)
    a = T.Append(gp, "f16", cache, seqs, 4, 2, 64, 64, "halves", 31)
    info = a.launch()
    assert info.total_tiles < info.shape[0]  # (claims, tiles)
    a.check()
    want = a.left()
    for limit in (1, 0):
        T.clean(a)
        flag = gp.Flag()
        st = gp.BlpState(1, flag, 32)
        a.launch(st.ctx(inject_at=1, max_workgroups=limit, poll_every=1))
        a.left()
        assert flag.get() == 1 and (limit == 0 or st.stop_index() == 0 and not T.same(a.left(), want))
        flag.set(0)
        st.clear_stop()
        a.launch(st.ctx(max_workgroups=limit, poll_every=1))
        assert T.same(a.left(), want)


@pytest.mark.parametrize("share", [0.1, 0.999])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [3, 9001, 140000])
def test_alternatives_among_many_nans(gp, dt, vocab, share):
    """signalling NaN for some or nearly all logits: the alternatives are what is left, also where that is fewer than are asked for"""
    ints, bad = {"f32": (torch.int32, 0x7F800001), "bf16": (torch.int16, 0x7F81)}[dt]
    rng = T.gen(40)
    x = torch.randn((3, vocab), generator=rng).to(S.TORCH[dt])
    x.view(ints)[torch.rand((3, vocab), generator=rng) < share] = bad
    x.view(ints)[:, 1] = bad
    a = T.Logprobs(gp, dt, x, torch.tensor([0, 1, 2]), 32)
    a.launch()
    got = a.left()
    assert torch.equal(got["ids"], S.logprobs(x, torch.zeros(3), 1.0, 32)[2])
    assert got["logprob"].isnan().all() and got["values"][got["ids"] >= 0].isnan().all() and (got["values"][got["ids"] < 0] == -torch.inf).all()
