"""Products with 4-bit weights, attention of sequences that begin alike, and attention over packed prompts, against their definitions in 64 bits."""
import math

import pytest
import torch

import serving as S
from test_serving_gpu import Append, Attend, Logprobs, bits, gen, same

pytestmark = pytest.mark.gpu
DTS = ["f16", "bf16"]
ACTS = {"none": lambda x: x, "relu": torch.relu, "gelu": torch.nn.functional.gelu}


# ---- 4-bit weights -------------------------------------------------------------------------------------------------------


class W4:
    """A call of gp_launch_gemm_w4, and what it has to leave; pad: elements between the rows of everything, which hold NaN (and C's sevens)"""

    def __init__(self, gp, dt, m, n, k, group, seed, zeros=True, bias=True, residual=True, act="none", pad=0, in_place=False, spread=16, change=None):
        self.gp, self.dt, self.m, self.n, self.k, self.group, self.act, self.in_place = gp, dt, m, n, k, group, act, in_place
        rng, t = gen(seed), S.TORCH[dt]
        groups = k // group

        def padded(x, by, fill):
            room = torch.full((x.shape[0], x.shape[1] + by), fill, dtype=x.dtype)
            room[:, : x.shape[1]] = x
            return room

        self.a = torch.randn((m, k), generator=rng).to(t)
        self.q = torch.randint(0, 16, (n, k), generator=rng, dtype=torch.uint8)
        self.scales = ((torch.rand((n, groups), generator=rng) + 0.5) * (torch.rand((n, groups), generator=rng) < 0.5).float().add(0.2) / 16).to(t)
        self.zeros = torch.randint(0, spread, (n, groups), generator=rng, dtype=torch.uint8) if zeros else None
        self.bias = torch.randn((n,), generator=rng).to(t) if bias else None
        self.residual = torch.randn((m, n), generator=rng).to(t) if residual else None
        if change:
            change(self)
        w = self.q[:, 0::2] | self.q[:, 1::2] << 4
        self.dev = {"a": padded(self.a, 8 * pad, math.nan).cuda(), "w": padded(w, 16 * pad, 0x77).cuda(), "scales": padded(self.scales, pad, math.nan).cuda(),
                    "zeros": padded(self.zeros, 3 * pad, 0xFF).cuda() if zeros else None, "bias": self.bias.cuda() if bias else None}
        self.before = padded(self.residual, pad, 7.0) if residual else None
        self.dev["residual"] = self.before.cuda() if residual else None
        self.c = self.dev["residual"].clone() if in_place else torch.full((m, n + pad), 7.0, dtype=t, device="cuda")
        d, at = self.dev, lambda x: None if x is None else x.data_ptr()
        self.p = gp.GemmW4Params(dtype=gp.DTYPE_BY_NAME[dt], M=m, N=n, K=k, group=group, A=at(d["a"]), lda=k + 8 * pad, W=at(d["w"]), ldw=k // 2 + 16 * pad, scales=at(d["scales"]),
                                 ld_scales=groups + pad, zeros=at(d["zeros"]), ld_zeros=groups + 3 * pad, C=at(self.c), ldc=n + pad, bias=at(d["bias"]),
                                 residual=at(self.c if in_place else d["residual"]), act={"none": gp.ACT_NONE, "relu": gp.ACT_RELU, "gelu": gp.ACT_GELU}[act])

    def launch(self, ctx=None, stream=None):
        return self.gp.launch("gp_launch_gemm_w4", self.p, ctx, stream)

    def clean(self):
        self.c.copy_(self.before) if self.in_place else self.c.fill_(7.0)
        torch.cuda.synchronize()

    def left(self):
        torch.cuda.synchronize()
        return self.c.cpu()

    def definition(self):
        """(the result, and the sum of what is added up, by magnitude) in 64 bits"""
        a, s = self.a.double(), self.scales.double().repeat_interleave(self.group, 1)
        z = 8.0 if self.zeros is None else self.zeros.double().repeat_interleave(self.group, 1)
        w, mass = (self.q.double() - z) * s, (self.q.double() + z) * s.abs()
        self.weight_mass = a.abs() @ w.abs().t().contiguous()
        y, mass = a @ w.t().contiguous(), a.abs() @ mass.t().contiguous()
        for x in (self.bias, self.residual):
            if x is not None:
                y, mass = y + x.double(), mass + x.double().abs()
        return ACTS[self.act](y), mass

    def check(self):
        got, (want, mass) = self.left(), self.definition()
        # one rounding to the type; in front of it sums in fp32: a group's values in turn, their sum and zero into the sum over the groups, wavefronts' sums,
        # each off by a unit at most.  (The activations are at most 1.13 times as steep, and off by a few units of their own.)
        deep = self.group + 2 * self.k // self.group + 32
        allowed = S.half_step(self.dt) * want.abs() + 1.13 * deep * 2.0 ** -23 * mass + (2.0 ** -25 if self.dt == "f16" else 0.0)
        if self.m > 128:  # many rows: W is rounded to the type in front of the products: each of them is off by half a unit of |a| |w|, and fp16's smallest by half of their step
            allowed += 1.13 * (S.half_step(self.dt) * self.weight_mass + (2.0 ** -25 if self.dt == "f16" else 0.0) * self.a.double().abs().sum(1, keepdim=True))
        err = (got[:, : self.n].double() - want).abs()
        # (from half a step above the type's largest on a value is rounded to infinity)
        border = float(torch.finfo(S.TORCH[self.dt]).max) * (1 + S.half_step(self.dt) / 2)
        err[(got[:, : self.n].double() == want.sign() * math.inf) & (want.abs() + allowed >= border)] = 0.0
        assert (err <= allowed).all(), (float((err / allowed).max()), (err / allowed).argmax())
        assert (got[:, self.n:] == 7.0).all()


W4S = [
    # m, n, k, group
    (1, 1, 32, 32), (1, 16, 128, 128), (1, 2304, 768, 64), (2, 17, 64, 64), (3, 33, 96, 32), (5, 129, 1056, 32), (15, 100, 640, 128), (16, 48, 192, 64),
    (17, 40, 448, 64), (31, 65, 1280, 128), (32, 7, 160, 32), (33, 100, 256, 64), (63, 130, 384, 128), (64, 32, 224, 32), (65, 257, 512, 128), (100, 31, 320, 64),
    (129, 130, 352, 32), (130, 300, 1152, 128), (200, 515, 576, 64), (257, 256, 256, 128),
    (2, 20, 32 * 300, 32), (20, 20, 64 * 258, 64), (40, 9, 32 * 513, 32),  # scales in several panels
    (3, 16400, 96, 32), (20, 16401, 160, 32), (50, 16400, 128, 64), (2, 65600, 128, 128),  # more rows of W to a wavefront
    (1101, 1303, 160, 32), (1101, 1303, 192, 64), (1100, 1302, 384, 128), (1025, 1281, 32, 32),  # tiles of 128 x 128
    (2945, 3001, 96, 32), (2945, 3001, 320, 64), (3000, 2945, 256, 128),  # ... of 128 x 256
]


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("case", range(len(W4S)))
def test_products_match_their_definition(gp, dt, case):
    m, n, k, group = W4S[case]
    w = W4(gp, dt, m, n, k, group, 10 + case, zeros=case % 3 != 0, bias=case % 2 == 0, residual=case % 4 < 2, act=list(ACTS)[case % 3], pad=case % 3, in_place=case % 4 == 1)
    w.launch()
    w.check()
    first = w.left()
    w.clean()
    w.launch()
    assert torch.equal(w.left(), first)


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m", [16, 48, 128, 384, 1100])
def test_every_number_is_where_it_belongs(gp, dt, group, m):
    """rows of A with a single one: a column of W each, exactly"""
    k = 384

    def one_hot(w):
        w.a.zero_()
        w.a[torch.arange(m), torch.arange(m) * 5 % k] = 1.0
    w = W4(gp, dt, m, 77 if m < 1000 else 1301, k, group, 3, bias=False, residual=False, spread=256, change=one_hot)
    w.launch()
    exact = ((w.q.double() - w.zeros.double().repeat_interleave(group, 1)) * w.scales.double().repeat_interleave(group, 1))[:, torch.arange(m) * 5 % k].t()
    assert torch.equal(w.left(), exact.to(S.TORCH[dt]))


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("m", [3, 40, 200, 1200])
def test_rows_of_large_and_of_no_size(gp, dt, m):
    """rows of zeros, of one sign and far from zero, of the type's smallest and of large values; a row with a NaN and one with an infinity, which nobody else sees"""
    def change(w):
        w.a[0] = 0.0
        w.a[1] += 30.0
        if m > 3:
            w.a[2] *= 2.0 ** -14
            w.a[3] = 4000.0
            w.a[m - 2, 17], w.a[m - 1, 5] = math.nan, math.inf
        w.scales[1], w.scales[2, 1] = 0.0, -0.5
        w.scales[3] *= 2.0 ** -9
    w = W4(gp, dt, m, 150 if m < 1000 else 1301, 512, 64, 5, residual=False, change=change)
    w.launch()
    got = w.left()
    if m > 3:
        assert not torch.isfinite(got[m - 2:]).any()
        w.a, w.c, w.m = w.a[: m - 2], w.c[: m - 2], m - 2
        w.residual = None
    w.check()


@pytest.mark.parametrize("m, n", [(3, 40), (200, 40), (1101, 1301)])
def test_weights_and_rows_behind_four_gigabytes(gp, m, n):
    """the last rows of W, A and C lie behind 2^32 bytes (2^31 elements); the bits of the same call close together"""
    small = W4(gp, "f16", m, n, 256, 128, 8, residual=False)
    small.launch()
    want = small.left()
    far = W4(gp, "f16", m, n, 256, 128, 8, residual=False)
    p = far.p
    ldw, ld = (1 << 32) // (n - 1) // 16 * 16 + 16, (1 << 32) // (m - 1) // 8 * 8 + 8
    ld = max(ld, (n + 7) // 8 * 8)
    w, a, c = (torch.empty(size, dtype=t, device="cuda") for size, t in ((ldw * (n - 1) + 128, torch.uint8), (ld * (m - 1) + 256, torch.half), (ld * (m - 1) + n, torch.half)))
    w.as_strided((n, 128), (ldw, 1)).copy_(far.dev["w"])
    a.as_strided((m, 256), (ld, 1)).copy_(far.dev["a"])
    p.W, p.ldw, p.A, p.lda, p.C, p.ldc = w.data_ptr(), ldw, a.data_ptr(), ld, c.data_ptr(), ld
    far.launch()
    torch.cuda.synchronize()
    assert torch.equal(c.as_strided((m, n), (ld, 1)).cpu(), want)


# ---- sequences that begin alike -------------------------------------------------------------------------------------------


def begin_alike(seqs, shared):
    """the first `shared` tokens of all sequences in the first one's pages"""
    seqs.table[:, : shared // seqs.page] = seqs.table[0, : shared // seqs.page].clone()
    seqs.shared = shared
    return seqs


class Prefix(Attend):
    """variant: None: together where that can be"""

    def __init__(self, gp, dt, cache_dtype, seqs, *args, variant=None, **kw):
        super().__init__(gp, dt, cache_dtype, seqs, *args, **kw)
        rows = seqs.max_new * self.heads // self.p.cache.kv_heads
        self.together = seqs.shared > 0 and rows <= 64
        if variant is None:
            variant = gp.PREFIX_TOGETHER if self.together else gp.PREFIX_AUTO
        self.shared_table = seqs.table[0, : seqs.shared // seqs.page].contiguous().cuda()
        self.prefix = gp.PrefixAttentionParams(attention=self.p, shared_len=seqs.shared, shared_table=self.shared_table.data_ptr() if seqs.shared else None,
                                               variant=variant)
        self.p = self.prefix.attention
        n = gp.C.c_size_t()
        gp.check(gp.lib().gp_prefix_attention_work_bytes(gp.C.byref(self.prefix), gp.C.byref(n)))
        self.work = torch.zeros(max(16, n.value), dtype=torch.uint8, device="cuda")
        self.p.work, self.p.work_bytes = self.work.data_ptr() if n.value else None, n.value

    def launch(self, ctx=None, stream=None):
        return self.gp.launch("gp_launch_prefix_attention", self.prefix, ctx, stream)

    def clean(self):
        self.out.fill_(7.0)
        torch.cuda.synchronize()


PREFIXES = [
    # lens, news, page, shared, heads, kv_heads, dim, causal
    ([65], None, 16, 64, 1, 1, 64, True),
    ([211, 260, 209], None, 16, 208, 12, 12, 64, True),
    ([700, 641, 1500, 650], None, 64, 640, 8, 2, 128, True),
    ([1030, 1024, 1025, 1200], None, 128, 1024, 24, 3, 128, True),  # one has nothing of its own but lies wholly in what is shared
    ([300, 100, 0, 290, 17], None, 32, 288, 8, 4, 64, True),        # some are shorter than what the others share
    ([330, 340, 7, 325, 300], [5, 4, 7, 0, 3], 32, 320, 6, 2, 128, True),
    ([530, 522, 514], [17, 9, 1], 64, 512, 9, 3, 64, False),
    ([200, 150, 20], [150, 150, 20], 64, 64, 4, 2, 128, True),      # rows in front of the shared tokens' end
    ([640 + 3 * i for i in range(33)], None, 64, 640, 4, 1, 64, True),   # more rows than a block
    ([200 + 70 * (i % 3) for i in range(150)], None, 16, 192, 4, 2, 64, True),
    ([210 + i % 7 for i in range(70)], [1 + i % 3 for i in range(70)], 16, 208, 8, 1, 64, True),
    ([400, 500, 700], None, 64, 0, 8, 2, 64, True),                 # nothing is shared
    ([2100, 2050], None, 128, 2048, 16, 1, 128, True),
    ([600, 700], [90, 70], 64, 512, 8, 2, 64, True),                # many rows of each
    ([1900, 1810, 1801], [8, 7, 8], 128, 1792, 8, 1, 128, True),    # 64 rows, the most that go together; seven parts
    ([800, 790, 781, 800, 770], [11, 4, 11, 1, 2], 16, 768, 8, 2, 128, True),  # 44 rows, two blocks of 32; three parts
    ([640 + 2600, 640 + 40, 640 + 1300, 640 + 1], None, 64, 640, 4, 2, 64, True),  # own keys in parts
    ([640 + 2600, 640 + 40, 640 + 1300], [6, 6, 5], 64, 640, 8, 2, 128, False),
]


@pytest.mark.parametrize("cache", ["same", "e4m3"])
@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("case", range(len(PREFIXES)))
def test_attention_behind_a_shared_beginning_matches_its_definition(gp, dt, cache, case):
    lens, news, page, shared, heads, kv_heads, dim, causal = PREFIXES[case]
    seqs = S.Sequences(lens, news, page, gen(case), width=max(-(-max(lens) // page), shared // page), tail=2 if news else 0)
    a = Prefix(gp, dt, dt if cache == "same" else cache, begin_alike(seqs, shared), heads, kv_heads, dim, causal, 400 + case, pad=8 * (case % 3), scale=-0.2 if case == 6 else None)
    a.launch()
    a.check()
    first = a.left()
    a.clean()
    a.launch()  # the workspace is as it was
    assert torch.equal(a.left(), first)


@pytest.mark.parametrize("case", [1, 3, 5, 8])
def test_for_each_sequence_as_if_nothing_were_shared(gp, case):
    lens, news, page, shared, heads, kv_heads, dim, causal = PREFIXES[case]
    seqs = begin_alike(S.Sequences(lens, news, page, gen(case), width=max(-(-max(lens) // page), shared // page)), shared)
    a = Prefix(gp, "bf16", "e4m3", seqs, heads, kv_heads, dim, causal, 450 + case, variant=gp.PREFIX_EACH)
    a.launch()
    a.check()
    b = Attend(gp, "bf16", "e4m3", seqs, heads, kv_heads, dim, causal, 450 + case)
    b.launch()
    assert torch.equal(a.left(), b.left())


def test_what_the_launcher_chooses(gp):
    """together where much is shared by many: more workgroups than sequences and heads; the result is what it is either way"""
    seqs = begin_alike(S.Sequences([2048 + 1 + i % 9 for i in range(40)], None, 128, gen(21)), 2048)
    a = Prefix(gp, "bf16", "bf16", seqs, 16, 8, 64, True, 22, variant=gp.PREFIX_AUTO)
    assert a.launch().total_tiles > 8 * 40
    a.check()
    first = a.left()
    a.prefix.variant = gp.PREFIX_TOGETHER
    a.clean()
    a.launch()
    assert torch.equal(a.left(), first)


@pytest.mark.parametrize("batch", [2, 40])
def test_shared_and_own_pages_that_are_not_there(gp, batch):
    holes = {(0, 1): -1, (0, 6): 10 ** 9, (1, 7): -7, (0, 9): -1}
    seqs = S.Sequences([150, 170] + [140 + i for i in range(batch - 2)], None, 16, gen(11), holes=holes)
    for cache in ("f16", "e4m3"):
        a = Prefix(gp, "f16", cache, begin_alike(seqs, 128), 8, 2, 64, True, 12)
        a.launch()
        a.check()


def test_a_shared_beginning_up_to_max_len_and_the_tables_width(gp):
    seqs = S.Sequences([300, 210, 330], None, 64, gen(13))
    for max_len in (256, 201, 64):
        a = Prefix(gp, "bf16", "bf16", begin_alike(seqs, 192), 8, 2, 128, True, 14, max_len=max_len)
        a.launch()
        a.check()


@pytest.mark.parametrize("cache", ["f16", "bf16", "e4m3"])
@pytest.mark.parametrize("batch", [2, 40])
def test_one_key_takes_everything_on_either_side(gp, cache, batch):
    """the shared part's largest score is far above or far below that of a sequence's own part"""
    dt = "bf16" if cache == "bf16" else "f16"
    seqs = S.Sequences([500 + 3 * i for i in range(batch)], None, 32, gen(15))
    a = Prefix(gp, dt, cache, begin_alike(seqs, 448), 8, 2, 64, False, 16, scale=-0.5, peak=6.0)
    a.launch()
    a.check()


@pytest.mark.parametrize("batch", [3, 40])
def test_shared_pages_with_scales_far_apart(gp, batch):
    seqs = S.Sequences([300 + i for i in range(batch)], None, 32, gen(17))
    a = Prefix(gp, "f16", "e4m3", begin_alike(seqs, 256), 4, 2, 64, False, 18)
    for page in range(seqs.pages):
        a.cache["v_scale"][page] = [2.0 ** -20, 1.0, 2.0 ** -33][page % 3] / 20
        a.cache["k_scale"][page] = [0.5, 2.0 ** -12, 0.3][page % 3]
    a.dev["k_scale"].copy_(a.cache["k_scale"])
    a.dev["v_scale"].copy_(a.cache["v_scale"])
    a.launch()
    a.check()


@pytest.mark.parametrize("cache", ["f16", "e4m3"])
@pytest.mark.parametrize("case", [([100, 37, 1], None), ([90, 100, 60], [7, 1, 3]), ([2, 0, 33] * 30, None)])
def test_sequences_that_end_in_front_of_what_nobody_has_written_yet(gp, cache, case):
    """the shared pages' last slots are no sequence's, and hold NaN"""
    for causal in (True, False):
        a = Prefix(gp, "f16", cache, begin_alike(S.Sequences(*case, 64, gen(31), width=3), 128), 8, 2, 64, causal, 32)
        a.launch()
        a.check()


@pytest.mark.parametrize("cache", ["f16", "e4m3"])
def test_what_is_not_finite_reaches_only_who_sees_it(gp, cache):
    """NaN among the shared keys and values from token 300 on; who has 300 tokens or fewer, or 300 at his new one, is as if it were not there"""
    seqs = begin_alike(S.Sequences([2000, 300, 299, 1950, 17, 0, 305, 310], [1, 1, 4, 2, 3, 0, 1, 11], 64, gen(33), width=32), 1920)
    for causal in (True, False):
        a = Prefix(gp, "f16", cache, seqs, 8, 2, 128, causal, 34)
        a.launch()
        finite = a.left()
        for pos in range(300, 1920):
            page, slot = seqs.place(0, pos)
            for name in ("k", "v"):
                a.dev[name].view(torch.uint8 if cache == "e4m3" else torch.int16)[page, :, slot] = 0x7F if cache == "e4m3" else 0x7FFF
        a.clean()
        a.launch()
        got = a.left()
        for b in range(seqs.batch):
            for row, pos in seqs.rows(b):
                if seqs.lens[b] <= 300:
                    assert torch.equal(got[row], finite[row]), (b, pos)
                elif (pos if causal else seqs.lens[b] - 1) >= 300:
                    assert got[row].isnan().all(), (b, pos)


def test_bounds_on_what_is_new_are_only_bounds(gp):
    """sequences with fewer new tokens than max_new, none among them, rows behind the last"""
    for news in ([1, 2, 0], [0, 0, 0]):
        seqs = S.Sequences([700, 650, 640], news, 64, gen(19), tail=3, max_new=5)
        a = Prefix(gp, "bf16", "e4m3", begin_alike(seqs, 640), 8, 2, 64, True, 20)
        a.launch()
        a.check()


# ---- packed prompts -----------------------------------------------------------------------------------------------------------


class Packed:
    def __init__(self, gp, dt, lens, heads, kv_heads, dim, causal, seed, scale=None, tail=0, max_len=None, pad=0, peak=1.0, gap=0, change=None):
        self.gp, self.dt, self.lens, self.heads, self.kv_heads, self.dim, self.causal = gp, dt, list(lens), heads, kv_heads, dim, causal
        rng = gen(seed)
        self.tokens, self.cols = sum(lens) + tail, (heads + 2 * kv_heads) * dim
        self.start = [sum(lens[:i]) for i in range(len(lens) + 1)]
        self.max_len = max(1, max(lens)) if max_len is None else max_len
        self.scale = dim ** -0.5 if scale is None else scale
        self.qkv = (peak * torch.randn((self.tokens, self.cols + pad), generator=rng)).to(S.TORCH[dt])
        self.qkv[self.tokens - tail:] = math.nan  # (rows of no sequence may hold anything)
        if change:
            change(self)
        self.dev, self.dev_start = self.qkv.cuda(), torch.tensor(self.start, dtype=torch.int32).cuda()
        self.out = torch.full((self.tokens, heads * dim + pad), 7.0, dtype=S.TORCH[dt], device="cuda")
        at, es = self.dev.data_ptr(), 2 * dim
        self.p = gp.PackedAttentionParams(dtype=gp.DTYPE_BY_NAME[dt], batch=len(lens), tokens=self.tokens, max_len=self.max_len, start=self.dev_start.data_ptr(), heads=heads, kv_heads=kv_heads,
                                          head_dim=dim, q=at, ld_q=self.cols + pad, k=at + es * heads, v=at + es * (heads + kv_heads), ld_kv=self.cols + pad, out=self.out.data_ptr(),
                                          ld_out=heads * dim + pad, scale=self.scale, causal=int(causal))

    def launch(self, ctx=None, stream=None):
        return self.gp.launch("gp_launch_packed_attention", self.p, ctx, stream)

    def clean(self):
        self.out.fill_(7.0)
        torch.cuda.synchronize()

    def left(self):
        torch.cuda.synchronize()
        return self.out.cpu()

    def check(self):
        got, cols, group = self.left(), self.heads * self.dim, self.heads // self.kv_heads
        written = torch.zeros(self.tokens, dtype=torch.bool)
        for r0, r1 in zip(self.start, self.start[1:]):
            n = min(r1 - r0, self.max_len)
            if n <= 0:
                continue
            written[r0: r0 + n] = True
            x = self.qkv[r0: r0 + n, : self.cols].double().view(n, -1, self.dim).transpose(0, 1)
            q, k, v = x[: self.heads], x[self.heads: self.heads + self.kv_heads].repeat_interleave(group, 0), x[self.heads + self.kv_heads:].repeat_interleave(group, 0)
            s = q @ k.transpose(1, 2).contiguous() * self.scale
            most = float((q.abs() @ k.abs().transpose(1, 2).contiguous()).max()) * abs(self.scale)
            if self.causal:
                s = s.masked_fill(torch.ones((n, n), dtype=torch.bool).triu(1), -math.inf)
            p = torch.softmax(s, -1)
            want, mass = p @ v, p @ v.abs()
            # as for the cache: probabilities and result are rounded to the type, a score is a sum of `dim` products in fp32
            half, score = S.half_step(self.dt), 2 * (self.dim + 8) * 2.0 ** -24 * max(most, 1.0)
            tiny = 2.0 ** -24 if self.dt == "f16" else 0.0
            y = got[r0: r0 + n, :cols].view(n, self.heads, self.dim).transpose(0, 1).double()
            allowed = half * (mass + want.abs()) + 2 * score * mass + tiny * (1 + mass.amax((0, 2), keepdim=True) * 64)
            err = (y - want).abs()
            assert (err <= allowed).all(), (r0, float((err / allowed).max()))
        assert (got[:, cols:] == 7.0).all() and (got[~written] == 7.0).all()


PACKEDS = [
    # lens, heads, kv_heads, dim, causal
    ([1], 1, 1, 64, True), ([2, 1, 3], 2, 1, 128, True), ([211], 12, 12, 64, True), ([63, 64, 65, 1, 0, 127, 128, 129], 4, 2, 64, True),
    ([100, 384, 17, 200], 12, 12, 64, False), ([300, 77, 33], 9, 3, 128, True), ([129, 500], 8, 1, 128, True), ([333, 0, 0, 260], 3, 1, 64, False), ([700, 1000], 8, 2, 128, True),
    ([1300, 30], 4, 4, 64, False), ([40] * 20, 7, 7, 128, True),
]


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("case", range(len(PACKEDS)))
def test_packed_attention_matches_its_definition(gp, dt, case):
    lens, heads, kv_heads, dim, causal = PACKEDS[case]
    a = Packed(gp, dt, lens, heads, kv_heads, dim, causal, 500 + case, tail=case % 3, pad=8 * (case % 2), scale=-0.2 if case == 5 else None)
    a.launch()
    a.check()


@pytest.mark.parametrize("dt", DTS)
def test_packed_attention_with_peaked_scores(gp, dt):
    for causal in (True, False):
        a = Packed(gp, dt, [300, 150], 4, 2, 128, causal, 520, scale=0.5, peak=6.0)
        a.launch()
        a.check()


def test_one_sequence_does_not_see_another(gp):
    """NaN and infinities in one of them, and in the rows behind the last"""
    def change(a):
        a.qkv[100:200] = math.nan
        a.qkv[150] = math.inf
    for causal in (True, False):
        for dt in DTS:
            a = Packed(gp, dt, [100, 100, 130], 4, 2, 64, causal, 521, tail=5, change=change)
            a.launch()
            got = a.left()
            assert got[100:200].isnan().any(1).all()
            b = Packed(gp, dt, [100, 100, 130], 4, 2, 64, causal, 521, tail=5)
            b.launch()
            b.check()
            want = b.left()
            assert torch.equal(got[:100], want[:100]) and torch.equal(got[200:], want[200:])


def test_starts_that_make_no_sense(gp):
    """rows in front of the first, behind the last, sequences that end before they begin, and more tokens than max_len: nothing is touched that is not there"""
    a = Packed(gp, "f16", [90, 50, 60], 4, 2, 64, True, 522)
    for start, max_len in (([0, 90, 140, 200], 64), ([-5, 90, 80, 300], 90), ([10, 10, 2 ** 31 - 1, -2 ** 31], 200), ([190, 200, 260, 270], 90), ([-2 ** 31, 2 ** 31 - 1, -1, 50], 200)):
        a.clean()
        a.p.max_len = a.max_len = max_len
        a.dev_start.copy_(torch.tensor(start, dtype=torch.int32))
        a.launch()
        got = a.left()
        written = torch.zeros(200, dtype=torch.bool)
        for r0, r1 in zip(start, start[1:]):
            if r0 >= 0:
                written[r0: max(r0, min(r1, r0 + max_len, 200))] = True
        assert torch.equal((got != 7.0).any(1), written), start


def test_packed_rows_behind_four_gigabytes(gp):
    a = Packed(gp, "bf16", [70, 60], 4, 2, 64, True, 523)
    a.launch()
    want = a.left()
    ld = (1 << 32) // 129 // 8 * 8 + 8
    far, out = (torch.empty(129 * ld + 8 * 64, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    for r in range(130):
        far[r * ld: r * ld + a.cols] = a.dev[r]
    at = far.data_ptr()
    a.p.q, a.p.k, a.p.v, a.p.ld_q, a.p.ld_kv, a.p.out, a.p.ld_out = at, at + 128 * 4, at + 128 * 6, ld, ld, out.data_ptr(), ld
    a.launch()
    torch.cuda.synchronize()
    for r in range(130):
        assert torch.equal(out[r * ld: r * ld + 256].cpu(), want[r]), r


# ---- stopped and resumed, other streams, graphs ----------------------------------------------------------------------------------


def calls(gp):
    got = [W4(gp, "bf16", 1, 300, 512, 128, 600), W4(gp, "f16", 20, 200, 384, 64, 601), W4(gp, "f16", 1100, 1300, 256, 32, 602, in_place=True, act="gelu"), W4(gp, "bf16", 3000, 2900, 256, 128, 603)]
    got.append(Prefix(gp, "f16", "f16", begin_alike(S.Sequences([2000, 1700, 1600], None, 64, gen(62)), 1536), 8, 4, 64, True, 63))
    got.append(Prefix(gp, "bf16", "e4m3", begin_alike(S.Sequences([900, 800, 1500], [3, 1, 4], 32, gen(64)), 768), 8, 4, 128, True, 65))
    got.append(Prefix(gp, "bf16", "bf16", begin_alike(S.Sequences([1300 + i for i in range(70)], None, 64, gen(66)), 1280), 8, 2, 64, True, 67))
    got.append(Packed(gp, "f16", [200, 300, 64, 1], 4, 2, 64, True, 68))
    got.append(Packed(gp, "bf16", [700, 5], 8, 2, 128, False, 69))
    return got


@pytest.mark.parametrize("which", range(9))
def test_stopped_and_resumed_has_the_bits_of_an_uninterrupted_launch(gp, which):
    call = calls(gp)[which]
    call.launch()
    want = call.left()
    for groups in (1, 32):
        flag = gp.Flag()
        st = gp.BlpState(1, flag, groups)
        call.clean()
        limit = 2 if groups == 1 else 0
        call.launch(st.ctx(inject_at=1, max_workgroups=limit, poll_every=1))
        call.left()
        assert flag.get() == 1
        if groups == 1:
            assert st.stop_index() == 0 and not same(call.left(), want)
        flag.set(0)
        st.clear_stop()
        call.launch(st.ctx(max_workgroups=limit, poll_every=1))
        assert same(call.left(), want), groups
    call.clean()
    call.launch()  # ... and the next launch finds its workspace as it needs it
    assert same(call.left(), want)


def test_two_streams_at_once(gp):
    first, second = calls(gp), calls(gp)
    want = []
    for c in first:
        c.launch()
        want.append(c.left())
        c.clean()
    streams = [gp.Stream(0), gp.Stream(1)]
    for _ in range(3):
        for a, b in zip(first, second):
            a.launch(stream=streams[0])
            b.launch(stream=streams[1])
        for s in streams:
            s.sync()
        for a, b, w in zip(first, second, want):
            assert same(a.left(), w) and same(b.left(), w)
            a.clean()
            b.clean()
    for s in streams:
        s.destroy()


def test_one_workspace_for_batches_of_any_sizes(gp):
    made = []
    for lens, news, shared, heads, kv_heads, dim in (([1500, 1400], None, 1280, 2, 2, 64), ([1500 + i for i in range(60)], None, 1408, 8, 4, 64), ([1700, 900, 1000], [1, 9, 3], 832, 16, 8, 128),
                                                     ([700 + i for i in range(5)], None, 640, 16, 16, 128), ([700 + i for i in range(300)], None, 640, 4, 4, 64), ([2600] * 8, [70] * 8, 640, 16, 2, 64), ([1500], None, 640, 2, 2, 64)):
        made.append(Prefix(gp, "bf16", "bf16", begin_alike(S.Sequences(lens, news, 64, gen(30)), shared), heads, kv_heads, dim, True, 31 + len(made)))
    room = max(c.p.work_bytes for c in made)
    work = torch.zeros(room, dtype=torch.uint8, device="cuda")
    want = []
    for c in made:
        c.launch()
        want.append(c.left())
        c.p.work, c.p.work_bytes = work.data_ptr(), room
    assert any(not c.together and c.p.work_bytes for c in made)
    for order in (made, made[::-1], made[::2] + made[1::2]):
        for c in order:
            c.clean()
            c.launch()
        for c, w in zip(made, want):
            assert torch.equal(c.left(), w)


def test_captured_and_replayed(gp):
    """in a graph, with other contents of the same buffers (lengths among them) every time and the program's own work in between"""
    stream = gp.Stream(0)
    seqs = begin_alike(S.Sequences([1800, 1500, 1540], None, 32, gen(70)), 1408)
    pre, pack, w4 = Prefix(gp, "bf16", "e4m3", seqs, 8, 4, 64, True, 72), Packed(gp, "bf16", [300, 200], 4, 2, 64, True, 73), W4(gp, "bf16", 3, 300, 512, 128, 74)
    made = (pre, pack, w4)
    for c in made:  # (what a first launch sets up is not part of the graph)
        c.launch(stream=stream)
    stream.sync()
    graph = gp.vp()
    gp.check(gp.lib().gp_graph_begin(stream.h))
    for c in made:
        c.launch(stream=stream)
    gp.check(gp.lib().gp_graph_end(stream.h, gp.C.byref(graph)))
    for i in range(4):
        pre.dev["kv_len"].copy_(torch.tensor([1800 - 90 * i, 1410 + i, 1540 - i], dtype=torch.int32))
        pre.dev["q"].copy_(torch.randn(pre.q.shape, generator=gen(80 + i)).bfloat16())
        pack.dev_start.copy_(torch.tensor([0, 300 - 40 * i, 500 - 50 * i], dtype=torch.int32))
        pack.dev.copy_(torch.randn(pack.qkv.shape, generator=gen(90 + i)).bfloat16())
        w4.dev["a"].copy_(torch.randn(w4.dev["a"].shape, generator=gen(95 + i)).bfloat16())
        for c in made:
            c.clean()
        gp.check(gp.lib().gp_graph_launch(graph, stream.h))
        stream.sync()
        got = [c.left() for c in made]
        for c in made:
            c.clean()
            c.launch()
        for g, c in zip(got, made):
            assert torch.equal(g, c.left()), (i, type(c))
    gp.check(gp.lib().gp_graph_destroy(graph))
    stream.destroy()


# ---- together -----------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
def test_users_behind_one_prompt(gp, cache):
    """A prompt is scored without a cache and put into one, then three users go on behind it for some steps: projection (4-bit weights), append, attention behind the shared
    prompt, projection back onto the residual, logits, log probabilities, on one stream; each against 64 bits from what the one in front of it has left."""
    dt, t = "bf16", torch.bfloat16
    heads, kv_heads, dim, page, width, vocab, prompt, users, steps = 8, 2, 64, 32, 256, 1000, 320, 3, 4
    rng, stream = gen(700), gp.Stream(0)
    cols, half = (heads + 2 * kv_heads) * dim, S.half_step(dt)
    inv_freq = (10000.0 ** (-torch.arange(0, dim, 2) / dim)).float()
    freq = inv_freq.cuda()

    def weights(n, k, group, seed):
        w = W4(gp, dt, 1, n, k, group, seed, bias=False, residual=False)
        w.scales *= 0.1
        w.dev["scales"].mul_(0.1)
        return w

    w_qkv, w_out, w_vocab = weights(cols, width, 64, 701), weights(width, heads * dim, 128, 702), weights(vocab, width, 32, 703)

    def project(w, a, residual=None):
        c = torch.empty((a.shape[0], w.n), dtype=t, device="cuda")
        p = type(w.p).from_buffer_copy(w.p)
        p.M, p.A, p.lda, p.C, p.ldc, p.residual = a.shape[0], a.data_ptr(), a.shape[1], c.data_ptr(), w.n, residual.data_ptr() if residual is not None else None
        torch.cuda.synchronize()
        gp.launch("gp_launch_gemm_w4", p, None, stream)
        stream.sync()
        w.m, w.a, w.residual, w.c = a.shape[0], a.cpu(), None if residual is None else residual.cpu(), c
        w.check()
        return c

    total = S.Sequences([prompt + steps] * users, None, page, gen(710))
    begin_alike(total, prompt)
    pool = S.cache_of(total, kv_heads, dim, cache, rng)
    dev = {n: x.cuda() for n, x in pool.items()}
    shared_table = total.table[0, : prompt // page].contiguous().cuda()
    work = None

    def sequences(lens, news, rows):
        s = S.Sequences(lens, news, page, gen(0), width=total.width)
        s.table, s.pages, s.shared = total.table[:rows], total.pages, prompt
        return s, {**s.device(), **dev}

    def append(s, d, qkv):
        q = torch.empty((s.tokens, heads * dim), dtype=t, device="cuda")
        at, es = qkv.data_ptr(), 2 * dim
        gp.launch("gp_launch_kv_append", gp.KvAppendParams(dtype=gp.BF16, cache=S.cache_params(gp, d, cache, kv_heads, dim, s), **S.sequence_params(s, d), heads=heads, q=at, k=at + es * heads,
                                                           v=at + es * (heads + kv_heads), ld_qkv=cols, q_out=q.data_ptr(), ld_q_out=heads * dim, inv_freq=freq.data_ptr(), rot_dim=dim,
                                                           rot_pairs=gp.ROT_HALVES), stream=stream)
        stream.sync()
        return q

    # the prompt: no cache is needed to score it (without positions, that is); then it goes into the pages that all share
    x = torch.randn((prompt, width), generator=rng).to(t).cuda()
    qkv = project(w_qkv, x)
    pack = Packed(gp, dt, [prompt], heads, kv_heads, dim, True, 1)
    pack.qkv = qkv.cpu()
    pack.dev.copy_(qkv)
    pack.launch(stream=stream)
    stream.sync()
    pack.check()
    project(w_vocab, project(w_out, pack.out, x))
    s, d = sequences([prompt], [prompt], 1)
    append(s, d, qkv)

    x = torch.randn((users, width), generator=rng).to(t).cuda()
    for step in range(steps):
        s, d = sequences([prompt + step + 1] * users, None, users)
        qkv = project(w_qkv, x)
        q = append(s, d, qkv)
        out = torch.empty_like(q)
        p = gp.PrefixAttentionParams(shared_len=prompt, shared_table=shared_table.data_ptr(), attention=gp.PagedAttentionParams(
            dtype=gp.BF16, cache=S.cache_params(gp, d, cache, kv_heads, dim, s), **S.sequence_params(s, d), heads=heads, max_len=prompt + steps, q=q.data_ptr(), ld_q=heads * dim,
            out=out.data_ptr(), ld_out=heads * dim, scale=0.125, causal=1))
        if work is None:
            n = gp.C.c_size_t()
            gp.check(gp.lib().gp_prefix_attention_work_bytes(gp.C.byref(p), gp.C.byref(n)))
            work = torch.zeros(max(16, n.value), dtype=torch.uint8, device="cuda")
            torch.cuda.synchronize()
        p.attention.work, p.attention.work_bytes = work.data_ptr(), work.numel()
        gp.launch("gp_launch_prefix_attention", p, None, stream)
        stream.sync()
        want, mass, most = S.attend(s, {n: x.cpu() for n, x in dev.items()}, q.cpu().view(users, heads, dim), 0.125, True)
        for row, ref in want.items():
            allowed = half * (mass[row] + ref.abs()) + 4 * (dim + 8) * 2.0 ** -24 * max(most, 1.0) * mass[row]
            assert ((out[row].cpu().view(heads, dim).double() - ref).abs() <= allowed).all()
        x = project(w_out, out, x)
        logits = project(w_vocab, x)
        lp = Logprobs(gp, dt, logits.cpu(), torch.arange(users), 4)
        lp.launch(stream=stream)
        stream.sync()
        lp.check()
    stream.destroy()


# ---- 4-bit weights: what is not finite, and one precision for all sizes ---------------------------------------------------------


EVERY_SIZE = [(3, 150, 512, 64), (40, 150, 512, 64), (200, 150, 512, 64), (1200, 1301, 512, 64), (1200, 1301, 512, 128), (1200, 1301, 544, 32), (65, 11009, 96, 32), (2945, 3001, 192, 64)]


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("m, n, k, group", EVERY_SIZE)
def test_what_is_not_finite_stays_so_behind_every_activation(gp, dt, act, m, n, k, group):
    """NaN and infinities in rows of A, among the scales, in bias and residual: a sum that is NaN comes out as NaN, one that is infinite as infinite or NaN (ReLU and GELU take minus infinity to 0)"""
    def change(w):
        w.a[0, 3] = math.nan
        w.a[1, 5], w.a[2, 5] = math.inf, -math.inf
        w.scales[7, 1], w.scales[8, 0] = math.nan, math.inf
        w.bias[9], w.bias[10], w.bias[11] = math.nan, math.inf, -math.inf
        w.residual[m - 1, 12], w.residual[m - 1, 13], w.residual[m - 1, 14] = math.nan, math.inf, -math.inf
    w = W4(gp, dt, m, n, k, group, 71, act=act, change=change)
    w.launch()
    got = w.left()[:, :n]
    w.act = "none"
    total, _ = w.definition()
    plain = torch.isfinite(total)
    assert torch.isfinite(got[plain]).all()
    assert got[total.isnan()].isnan().all() and got[:, 8].isnan().all()
    up, down = got[total == math.inf], got[total == -math.inf]
    assert (up.isnan() | (up == math.inf)).all()
    assert (down.isnan() | (down == (-math.inf if act == "none" else 0.0)) | ((down == -math.inf) if act == "gelu" else False)).all()
    assert (total == math.inf).any() and (total == -math.inf).any() and total.isnan().any()


class ExactW4(W4):
    """... whatever the size: nothing but the result is rounded to 16 bits"""

    def check(self):
        got, (want, mass) = self.left(), self.definition()
        deep = self.group + 2 * self.k // self.group + 32
        allowed = S.half_step(self.dt) * want.abs() + 1.13 * deep * 2.0 ** -23 * mass + (2.0 ** -25 if self.dt == "f16" else 0.0)
        err = (got[:, : self.n].double() - want).abs()
        assert (err <= allowed).all(), (float((err / allowed).max()), (err / allowed).argmax())
        assert (got[:, self.n:] == 7.0).all()


EXACT = [
    (65, 11009, 96, 32), (100, 11009, 256, 128), (128, 23000, 192, 64),  # one tile of rows, partly empty, of many columns
    (129, 130, 352, 32), (130, 300, 1152, 128), (200, 515, 576, 64), (257, 256, 256, 128),
    (1101, 1303, 160, 32), (1101, 1303, 192, 64), (1100, 1302, 384, 128), (1025, 1281, 32, 32), (700, 2000, 2048, 128), (2945, 3001, 96, 32), (2945, 3001, 320, 64), (3000, 2945, 256, 128),
]


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("case", range(len(EXACT)))
def test_only_the_result_is_rounded_whatever_the_size(gp, dt, case):
    m, n, k, group = EXACT[case]
    w = ExactW4(gp, dt, m, n, k, group, 500 + case, zeros=case % 3 != 0, bias=case % 2 == 0, residual=case % 4 < 2, act=list(ACTS)[case % 3], pad=case % 3, in_place=case % 4 == 1, spread=256 if case % 2 else 16)
    w.launch()
    w.check()
    first = w.left()
    w.clean()
    w.launch()
    assert torch.equal(w.left(), first)


@pytest.mark.parametrize("m, n", [(3, 150), (200, 150), (1200, 1301)])
def test_weights_beyond_the_largest_of_16_bits(gp, m, n):
    """fp16: a scale of 8000 times numbers up to 15 less 0: weights up to 120000, sums that fit"""
    def change(w):
        w.a *= 2.0 ** -9
        w.scales[5], w.zeros[5] = 8000.0, 0
    w = ExactW4(gp, "f16", m, n, 256, 64, 73, bias=False, residual=False, change=change)
    assert float((w.q[5].double() * 8000).max()) > 65504
    w.launch()
    w.check()


def test_rows_are_as_exact_among_many_as_alone(gp):
    many = ExactW4(gp, "bf16", 1200, 1301, 512, 64, 74)
    for m in (1, 40, 1200):
        w = ExactW4(gp, "bf16", m, 1301, 512, 64, 75, change=lambda w: [getattr(w, x).copy_(getattr(many, x)[: m] if x in ("a", "residual") else getattr(many, x)) for x in ("a", "residual", "q", "scales", "zeros", "bias")])
        w.launch()
        w.check()


# ---- sequences that end within a long shared beginning ----------------------------------------------------------------------------


def long_beginning(lens, news, page, shared, rng):
    """as begin_alike, without pages in the pool that nobody names"""
    seqs = S.Sequences(lens, news, page, rng, width=max(1, -(-(max(lens) - shared) // page)))
    pages = shared // page
    seqs.table = torch.cat([torch.arange(seqs.pages, seqs.pages + pages, dtype=torch.int32).repeat(seqs.batch, 1), seqs.table], 1)
    seqs.pages, seqs.width, seqs.shared = seqs.pages + pages, seqs.width + pages, shared
    return seqs


LONG_BEGINNINGS = [
    # lens, news, page, shared, heads, kv_heads, dim: keys of a sequence that does not see all of what is shared are more than a tile's
    ([16384 + 9 + i for i in range(6)] + [16000, 9000, 16384, 1, 0], None, 128, 16384, 8, 2, 64),
    ([8192 + 40 + 3 * i for i in range(8)] + [8190, 8192 + 2, 5000], [3] * 8 + [3, 5, 1], 64, 8192, 8, 2, 64),  # one has new tokens in front of the end of what is shared
    ([4096 + 17] * 64 + [4000, 3999, 17] + [4096 + 2] * 3, None, 128, 4096, 8, 8, 64),  # many sequences, and parts of several of them
    ([4096 + 17] * 64 + [4095] * 6, [2] * 70, 128, 4096, 64, 8, 64),
    ([8192 + 700, 8192 + 30, 8000], None, 128, 8192, 8, 1, 128),  # own keys in parts anyway
    ([3000, 2999], None, 128, 4096, 8, 1, 128),  # nobody sees all of it
]


@pytest.mark.parametrize("cache", ["same", "e4m3"])
@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("case", range(len(LONG_BEGINNINGS)))
def test_sequences_that_end_within_a_long_beginning(gp, dt, cache, case):
    lens, news, page, shared, heads, kv_heads, dim = LONG_BEGINNINGS[case]
    a = Prefix(gp, dt, dt if cache == "same" else cache, long_beginning(lens, news, page, shared, gen(80 + case)), heads, kv_heads, dim, True, 600 + case)
    a.launch()
    a.check()
    first = a.left()
    a.clean()
    a.launch()
    assert torch.equal(a.left(), first)


def test_a_sequence_that_ends_within_a_long_beginning_is_not_left_to_one_workgroup(gp):
    """its 256 units of keys in one tile took 20 times what the others' call takes"""
    def took(lens):
        a = Prefix(gp, "bf16", "bf16", long_beginning(lens, None, 128, 32768, gen(90)), 4, 1, 64, True, 91)
        times = []
        for _ in range(9):
            begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            begin.record()
            for _ in range(20):
                a.launch()
            end.record()
            torch.cuda.synchronize()
            times.append(begin.elapsed_time(end))
        return sorted(times)[4]
    assert took([32768 + 20 + i for i in range(5)] + [32700]) < 6 * took([32768 + 20 + i for i in range(6)])


def test_what_nobody_sees_is_not_read_for_all(gp):
    """max_len, or the table, ends in front of the end of what is shared: each sequence for itself, whoever asks"""
    seqs = begin_alike(S.Sequences([300, 210, 330], None, 64, gen(13)), 192)
    for max_len, tiles in ((191, 3), (192, None)):
        a = Prefix(gp, "bf16", "bf16", seqs, 8, 2, 128, True, 14, max_len=max_len)
        got = a.launch().total_tiles
        assert (got == 2 * 3) if tiles else got >= 16
        a.check()


# ---- claims through several counters ----------------------------------------------------------------------------------------------


@pytest.mark.parametrize("which", range(5))
def test_claims_through_counters_have_the_bits_of_a_plain_launch(gp, which):
    """fewer workgroups than tiles, which claim through 16, 32 and 64 counters, whole and stopped and resumed"""
    call = [lambda: Prefix(gp, "bf16", "e4m3", begin_alike(S.Sequences([1300 + i for i in range(70)], None, 64, gen(92)), 1280), 8, 2, 128, True, 93),
            lambda: Prefix(gp, "f16", "f16", begin_alike(S.Sequences([2060, 2100, 1500, 2049] * 8, [2, 1, 3, 1] * 8, 64, gen(94), width=33), 2048), 16, 4, 64, True, 95),
            lambda: Packed(gp, "bf16", [2000, 700, 5, 1300], 8, 2, 64, True, 96),
            lambda: Packed(gp, "f16", [100 + 7 * i for i in range(30)], 4, 4, 128, False, 97),
            lambda: Attend(gp, "bf16", "e4m3", S.Sequences([900, 1800, 400], [900, 1500, 300], 64, gen(98)), 8, 2, 128, True, 99)][which]()
    clean = getattr(call, "clean", lambda: call.out.fill_(7.0))
    call.launch()
    want = call.left()
    for groups in (16, 32, 64):
        flag = gp.Flag()
        st = gp.BlpState(1, flag, groups)
        clean()
        info = call.launch(st.ctx(max_workgroups=64))
        assert info.total_tiles > info.grid  # claims go through the counters
        assert same(call.left(), want), groups
        st.reset()
        clean()
        call.launch(st.ctx(inject_at=groups, max_workgroups=64, poll_every=1))
        call.left()
        assert flag.get() == 1
        flag.set(0)
        st.clear_stop()
        call.launch(st.ctx(max_workgroups=64, poll_every=1))
        assert same(call.left(), want), groups


def test_many_sequences_of_which_some_end_within_a_long_beginning(gp):
    """more sequences than a workgroup's threads look at together, the ones that end early among the last, the first, or nobody"""
    seqs = long_beginning([2560 + 3 + i % 5 for i in range(600)], None, 128, 2560, gen(100))
    a = Prefix(gp, "f16", "f16", seqs, 1, 1, 64, True, 101)
    whole = None
    for early in ([], [599], [0, 255, 256, 300, 598]):
        lens = list(seqs.lens)
        for b in early:
            seqs.lens[b] = 2500 - b
        a.dev["kv_len"].copy_(torch.tensor(seqs.lens, dtype=torch.int32))
        a.clean()
        a.launch()
        if early == [599]:  # nobody else's result changes
            assert torch.equal(a.left()[:599], whole[:599]) and not torch.equal(a.left()[599], whole[599])
        else:
            a.check()
        whole = a.left()
        seqs.lens = lens
