"""The serving step's kernels at the borders of what they take: scales, NaN, probabilities and lengths (definitions and callers: serving.py, test_serving_gpu.py)."""
import pytest
import torch

import serving as S
import test_serving_gpu as T

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", ["bf16"])
def test_append_to_a_page_whose_scale_attention_takes_as_a_border(gp, dt):
    """8 bits: what append keeps, rescales and writes reads back on the scale that attention takes, 2^-60 .. 2^60, whatever scale the page came with or its values ask for"""
    lens, page, dim = [5, 5, 5, 5, 1], 16, 64
    seqs = S.Sequences(lens, None, page, T.gen(1))
    sizes = [0.0, 2.0 ** -64, 2.0 ** 62, 1.0, 2.0 ** 75]  # of the new tokens
    before = [2.0 ** -130, 2.0 ** -70, 2.0 ** 70, 2.0 ** -126, 1.0]  # the scales of their pages (the last one begins)

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
