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
