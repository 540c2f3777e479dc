"""A decoder's serving step (append to a paged cache, attention over it, log probabilities) against its definition in 64 bits."""
import math

import pytest
import torch

import serving as S

pytestmark = pytest.mark.gpu
DTS = ["f16", "bf16"]


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ---- append ----------------------------------------------------------------------------------------------------------


class Append:
    """A call of gp_launch_kv_append on packed q, k, v, and what it has to leave"""

    def __init__(self, gp, dt, cache_dtype, seqs, heads, kv_heads, dim, rot, pairs, seed, size=1.0, q=True, pad=0, base=10000.0, change=None):
        self.gp, self.dt, self.cache_dtype, self.seqs, self.heads, self.kv_heads, self.dim, self.rot, self.pairs = gp, dt, cache_dtype, seqs, heads, kv_heads, dim, rot, pairs
        rng = gen(seed)
        self.cache = S.cache_of(seqs, kv_heads, dim, cache_dtype, rng)
        self.qkv = (size * torch.randn((seqs.tokens, (heads + 2 * kv_heads) * dim + pad), generator=rng)).to(S.TORCH[dt])
        if change:
            change(self)
        self.inv_freq = (base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / max(rot, 1))).float()
        self.dev = {**seqs.device(), **{n: x.cuda() for n, x in self.cache.items()}, "qkv": self.qkv.cuda(), "inv_freq": self.inv_freq.cuda()}
        self.q_out = torch.full((seqs.tokens, heads * dim + pad), 7.0, dtype=S.TORCH[dt], device="cuda")
        at, es = self.dev["qkv"].data_ptr(), 2 * dim
        self.p = gp.KvAppendParams(dtype=gp.DTYPE_BY_NAME[dt], cache=S.cache_params(gp, self.dev, cache_dtype, kv_heads, dim, seqs), **S.sequence_params(seqs, self.dev), heads=heads,
                                   q=at if q else None, k=at + es * heads, v=at + es * (heads + kv_heads), ld_qkv=self.qkv.shape[1], q_out=self.q_out.data_ptr() if q else None,
                                   ld_q_out=self.q_out.shape[1], inv_freq=self.dev["inv_freq"].data_ptr() if rot else None, rot_dim=rot,
                                   rot_pairs=gp.ROT_HALVES if pairs == "halves" else gp.ROT_NEIGHBOURS)

    def part(self, first, n):
        return self.qkv[:, first * self.dim: (first + n) * self.dim].reshape(self.seqs.tokens, n, self.dim)

    def launch(self, ctx=None, stream=None):
        return self.gp.launch("gp_launch_kv_append", self.p, ctx, stream)

    def left(self):
        torch.cuda.synchronize()
        return {n: self.dev[n].cpu() for n in self.cache} | {"q": self.q_out.cpu()}

    def check(self):
        seqs, got = self.seqs, self.left()
        k, v, q = self.part(self.heads, self.kv_heads), self.part(self.heads + self.kv_heads, self.kv_heads), self.part(0, self.heads)
        want, scales, written, again = S.append(seqs, self.cache, self.cache_dtype, k, v, self.rot, self.pairs, self.inv_freq)
        # a pair's sum in fp32 behind products with cosines that are off by a millionth
        near = 4e-6 * float(self.qkv.double()[torch.isfinite(self.qkv)].abs().max()) * 2
        half = S.half_step(self.dt)
        tiny = 2.0 ** -25 if self.dt == "f16" else 0.0  # half a step of fp16's smallest values
        for name in ("k", "v"):
            x, ref = got[name], want[name]
            at = written[:, None, :, None].expand_as(x)
            if self.cache_dtype == "e4m3":
                assert torch.equal(got[name + "_scale"].double(), scales[name]), name
                for n, page, h in again:
                    if n == name:
                        rest = ~written[page]
                        old, new = ref[page, h, rest], x[page, h, rest].double()
                        fine = ~old.isnan()
                        assert torch.equal(new.isnan(), old.isnan())
                        assert ((new - old).abs() <= torch.maximum(2.0 ** -4 * old.abs(), torch.tensor(2.0 ** -10)))[fine].all(), (n, page, h)
                        at = at.clone()
                        at[page, h] = True
                err = (x.double() - ref).abs()
                allowed = torch.maximum(2.0 ** -4 * ref.abs(), torch.tensor(2.0 ** -10)) + (near / scales[name])[:, :, None, None]
                assert torch.equal(x.double().isnan()[at], ref.isnan()[at])
                assert (err <= allowed)[at & ~ref.isnan()].all(), name
                bits, old = x.view(torch.uint8), self.cache[name].view(torch.uint8)
            else:
                fine = at & torch.isfinite(ref)
                assert ((x.double() - ref).abs() <= half * ref.abs() + (near if name == "k" and self.rot else 0.0) + tiny)[fine].all(), name
                assert torch.isfinite(x.double()[fine]).all()
                bits, old = x.view(torch.int16), self.cache[name].view(torch.int16)
            assert torch.equal(bits[~at], old[~at]), name  # nothing else has changed
        rows = {row: pos for b in range(seqs.batch) for row, pos in seqs.rows(b)}
        for row in range(seqs.tokens):
            if row in rows and self.p.q:
                ref = S.turned(q[row].double(), rows[row], self.inv_freq, self.rot, self.pairs).flatten()
                x = got["q"][row, : self.heads * self.dim].double()
                fine = torch.isfinite(ref)
                assert ((x - ref).abs() <= half * ref.abs() + (near if self.rot else 0.0) + tiny)[fine].all(), row
                assert (got["q"][row, self.heads * self.dim:] == 7.0).all()
            else:
                assert (got["q"][row] == 7.0).all(), row


APPENDS = [
    # lens, news (None: one each), page, heads, kv_heads, dim, rot, pairs
    ([1], None, 16, 1, 1, 64, 64, "halves"),
    ([211, 16, 17, 1, 33], None, 16, 12, 12, 64, 64, "neighbours"),
    ([64, 65, 128, 1, 200], None, 64, 8, 2, 128, 128, "halves"),
    ([40, 130, 7, 0, 300], [17, 130, 7, 0, 65], 32, 6, 2, 128, 64, "neighbours"),
    ([200, 129], [71, 128], 128, 3, 1, 64, 32, "halves"),
    ([513], [513], 64, 4, 4, 128, 0, "halves"),
    ([5, 3], [3, 5], 16, 2, 1, 64, 16, "halves"),  # two of the second's tokens are in front of position 0
]


@pytest.mark.parametrize("cache", ["same", "e4m3"])
@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append_matches_its_definition(gp, dt, cache, case):
    lens, news, page, heads, kv_heads, dim, rot, pairs = APPENDS[case]
    seqs = S.Sequences(lens, news, page, gen(case), tail=2 if news else 0)
    a = Append(gp, dt, dt if cache == "same" else cache, seqs, heads, kv_heads, dim, rot, pairs, 100 + case, pad=8 * (case % 2))
    a.launch()
    a.check()


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
def test_append_drops_what_has_no_place(gp, cache):
    """pages that are not in the pool, entries past the table, and more new tokens than the call allows for"""
    holes = {(0, 1): -1, (1, 0): 2 ** 31 - 1, (2, 2): -2 ** 31}
    seqs = S.Sequences([40, 35, 90, 33], [40, 20, 70, 33], 16, gen(3), width=3, holes=holes, max_new=64, tail=1)
    a = Append(gp, "bf16", cache, seqs, 4, 2, 64, 64, "halves", 5)
    a.launch()
    a.check()


def test_append_far_positions(gp):
    """the angle of a position of two million, at frequencies from 1 down"""
    page, seqs = 128, S.Sequences([128], None, 128, gen(0))
    seqs.width = 2 ** 21 // page
    seqs.table = torch.full((1, seqs.width), -1, dtype=torch.int32)
    seqs.table[0, -1] = 1
    seqs.lens = [2 ** 21]
    a = Append.__new__(Append)
    seqs_len, seqs.lens = seqs.lens, [0]  # (nothing older is in the pool)
    Append.__init__(a, gp, "f16", "f16", seqs, 2, 1, 128, 128, "halves", 1)
    seqs.lens = seqs_len
    a.dev["kv_len"].fill_(2 ** 21)
    a.launch()
    a.check()


def test_append_scales_rise(gp):
    """8 bits: larger tokens come to a page that holds smaller ones (their values are rounded anew), smaller ones come to one with a large scale (nothing
    else changes), a page begins with zeros, infinities and NaN among the new values"""
    seqs = S.Sequences([20, 20, 17, 30, 16], [3, 3, 1, 14, 16], 16, gen(1))

    def change(a):
        a.cache["k_scale"][:], a.cache["v_scale"][:] = 2.0 ** -9, 0.75
        x = a.part(a.heads, 2 * a.kv_heads)
        rows = a.qkv.view(a.seqs.tokens, -1, 64)
        assert x.shape[1] == 4 and rows.shape[1] == 6
        rows[0:3, 2:] *= 1000.0
        rows[3:6, 2:] *= 2.0 ** -10
        rows[6, 2:] = 0.0
        rows[7, 4, 5], rows[8, 4, 6], rows[9, 4, 7] = math.inf, -math.inf, math.nan  # (the values, which are not rotated)

    a = Append(gp, "bf16", "e4m3", seqs, 2, 2, 64, 64, "halves", 9, change=change)
    a.launch()
    a.check()
    left = a.left()
    page = int(seqs.table[2, 1])
    assert (left["k_scale"][page] == S.LOWEST).all() and (left["k"][page, :, 0].float() == 0).all()
    page = int(seqs.table[3, 1])
    assert left["v"][page, 0, 0, 5].float() == 448 and left["v"][page, 0, 1, 6].float() == -448 and left["v"][page, 0, 2, 7].float().isnan()


def test_append_without_queries_and_in_place(gp):
    seqs = S.Sequences([40, 9], [21, 9], 32, gen(2))
    a = Append(gp, "f16", "f16", seqs, 3, 3, 64, 64, "halves", 4, q=False)
    a.launch()
    a.check()
    b, c = (Append(gp, "f16", "f16", seqs, 3, 3, 64, 64, "halves", 4) for _ in range(2))
    b.launch()
    c.p.q_out, c.p.ld_q_out = c.p.q, c.p.ld_qkv
    c.launch()
    torch.cuda.synchronize()
    assert torch.equal(c.dev["qkv"][:, : 3 * 64], b.q_out)
    assert torch.equal(c.dev["qkv"][:, 3 * 64:], b.dev["qkv"][:, 3 * 64:])
    assert torch.equal(c.dev["k"].view(torch.int16), b.dev["k"].view(torch.int16))


def test_append_again_changes_nothing(gp):
    """the same call twice leaves the same bits: the scales of the first fit"""
    seqs = S.Sequences([100, 64, 130], [37, 1, 100], 64, gen(6))
    a = Append(gp, "bf16", "e4m3", seqs, 4, 2, 128, 128, "neighbours", 7, size=50.0)
    a.launch()
    first = a.left()
    a.launch()
    second = a.left()
    assert all(torch.equal(first[n].view(torch.uint8), second[n].view(torch.uint8)) for n in first)


# ---- attention -----------------------------------------------------------------------------------------------------------


class Attend:
    def __init__(self, gp, dt, cache_dtype, seqs, heads, kv_heads, dim, causal, seed, scale=None, max_len=None, pad=0, peak=1.0):
        self.gp, self.dt, self.seqs, self.heads, self.dim, self.causal = gp, dt, seqs, heads, dim, causal
        rng = gen(seed)
        self.cache = S.cache_of(seqs, kv_heads, dim, cache_dtype, rng)
        if cache_dtype == "e4m3":  # keys of about the size that activations have
            self.cache["k_scale"] *= 0.05
        self.q = (peak * torch.randn((seqs.tokens, heads * dim + pad), generator=rng)).to(S.TORCH[dt])
        self.scale = dim ** -0.5 if scale is None else scale
        self.max_len = max_len
        self.dev = {**seqs.device(), **{n: x.cuda() for n, x in self.cache.items()}, "q": self.q.cuda()}
        self.out = torch.full((seqs.tokens, heads * dim + pad), 7.0, dtype=S.TORCH[dt], device="cuda")
        self.p = gp.PagedAttentionParams(dtype=gp.DTYPE_BY_NAME[dt], cache=S.cache_params(gp, self.dev, cache_dtype, kv_heads, dim, seqs), **S.sequence_params(seqs, self.dev),
                                         heads=heads, max_len=max(1, max(seqs.lens)) if max_len is None else max_len, q=self.dev["q"].data_ptr(), ld_q=self.q.shape[1],
                                         out=self.out.data_ptr(), ld_out=self.out.shape[1], scale=self.scale, causal=int(causal))
        self.workspace()

    def workspace(self):
        gp, n = self.gp, self.gp.C.c_size_t()
        gp.check(gp.lib().gp_paged_attention_work_bytes(gp.C.byref(self.p), gp.C.byref(n)))
        self.work = torch.zeros(max(16, n.value), dtype=torch.uint8, device="cuda")
        self.p.work, self.p.work_bytes = self.work.data_ptr() if n.value else None, n.value

    def launch(self, ctx=None, stream=None):
        return self.gp.launch("gp_launch_paged_attention", self.p, ctx, stream)

    def left(self):
        torch.cuda.synchronize()
        return self.out.cpu()

    def check(self):
        got, cols = self.left(), self.heads * self.dim
        q = self.q[:, :cols].reshape(self.seqs.tokens, self.heads, self.dim)
        want, mass, most = S.attend(self.seqs, self.cache, q, self.scale, self.causal, self.max_len)
        # the probabilities and the result are rounded to the type; a score is a sum of `dim` products in fp32, and its exponential and what
        # is summed afterwards are off by a few units of fp32
        half, score = S.half_step(self.dt), 2 * (self.dim + 8) * 2.0 ** -24 * max(most, 1.0)
        tiny = 2.0 ** -24 if self.dt == "f16" else 0.0  # a step of fp16's smallest values, of probabilities and of the result
        for row in range(self.seqs.tokens):
            x = got[row, :cols].reshape(self.heads, self.dim).double()
            if row not in want:
                assert (got[row] == 7.0).all(), row
                continue
            allowed = half * (mass[row] + want[row].abs()) + 2 * score * mass[row] + tiny * (1 + mass[row].amax() * 64)
            err = (x - want[row]).abs()
            assert (err <= allowed).all(), (row, float((err / allowed).max()))
            assert (got[row, cols:] == 7.0).all()


ATTENDS = [
    # lens, news, page, heads, kv_heads, dim, causal
    ([1], None, 16, 1, 1, 64, True),
    ([211, 16, 17, 0, 33, 1], None, 16, 12, 12, 64, True),
    ([700, 65, 1500, 1], None, 64, 8, 2, 128, True),
    ([3000], None, 128, 24, 1, 128, True),  # one head of the cache for more rows than a matrix instruction has
    ([300, 77, 33], None, 32, 9, 3, 64, True),
    ([130, 40, 7, 2, 300], [5, 4, 7, 0, 3], 32, 6, 2, 128, True),
    ([200, 150, 20], [150, 150, 20], 64, 4, 2, 128, True),
    ([333, 260], [129, 260], 16, 3, 1, 64, True),
    ([5, 3, 0], [3, 5, 2], 16, 2, 1, 64, True),  # rows that see nothing
    ([90, 1, 384, 0], [33, 70, 5, 4], 64, 4, 4, 64, False),  # another sequence's states
    ([1000], [3], 128, 8, 8, 128, False),
    ([600, 511], [290, 400], 128, 8, 1, 128, True),
]


@pytest.mark.parametrize("cache", ["same", "e4m3"])
@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("case", range(len(ATTENDS)))
def test_attention_matches_its_definition(gp, dt, cache, case):
    lens, news, page, heads, kv_heads, dim, causal = ATTENDS[case]
    seqs = S.Sequences(lens, news, page, gen(case), tail=2 if news else 0)
    a = Attend(gp, dt, dt if cache == "same" else cache, seqs, heads, kv_heads, dim, causal, 200 + case, pad=8 * (case % 3))
    a.launch()
    a.check()
    first = a.left()
    a.launch()  # the workspace is as it was
    assert torch.equal(a.left(), first)


@pytest.mark.parametrize("news", [None, [40, 70, 1]])
@pytest.mark.parametrize("cache", ["f16", "e4m3"])
def test_attention_leaves_out_pages_that_are_not_there(gp, cache, news):
    holes = {(0, 0): -1, (0, 3): 10 ** 9, (1, 1): -7, (2, 0): -1, (2, 1): -1, (2, 2): -1, (2, 3): -1, (2, 4): -1}
    seqs = S.Sequences([150, 170, 90], news, 32, gen(11), width=5, holes=holes)  # the second's last tokens are past the table
    a = Attend(gp, "f16", cache, seqs, 4, 2, 64, True, 12)
    a.launch()
    a.check()


@pytest.mark.parametrize("news", [None, [33, 80]])
def test_attention_up_to_max_len(gp, news):
    seqs = S.Sequences([300, 210], news, 64, gen(13))
    a = Attend(gp, "bf16", "bf16", seqs, 4, 2, 128, True, 14, max_len=201)
    a.launch()
    a.check()


@pytest.mark.parametrize("cache", ["f16", "bf16", "e4m3"])
@pytest.mark.parametrize("news", [None, [64, 100]])
def test_attention_with_peaked_scores(gp, cache, news):
    """one key takes everything, at either end of the sequence; negative scale"""
    dt = "bf16" if cache == "bf16" else "f16"
    seqs = S.Sequences([500, 357], news, 64, gen(15))
    a = Attend(gp, dt, cache, seqs, 4, 2, 128, False, 16, scale=-0.5, peak=6.0)
    a.launch()
    a.check()


@pytest.mark.parametrize("news", [None, [64, 100]])
def test_attention_with_scales_far_apart(gp, news):
    """pages whose values are millions of times smaller or larger than their neighbours', and the small ones are what is attended to"""
    seqs = S.Sequences([300, 357], news, 32, gen(17))
    a = Attend(gp, "f16", "e4m3", seqs, 4, 2, 64, False, 18)
    for b in range(2):
        for i in range(seqs.width):
            page = int(seqs.table[b, i])
            a.cache["v_scale"][page] = [2.0 ** -20, 1.0, 2.0 ** -33][i % 3] / 20
            a.cache["k_scale"][page] = [0.5, 2.0 ** -12, 0.3][i % 3]
    a.dev["k_scale"].copy_(a.cache["k_scale"])
    a.dev["v_scale"].copy_(a.cache["v_scale"])
    a.launch()
    a.check()


@pytest.mark.parametrize("cache", ["f16", "e4m3"])
@pytest.mark.parametrize("news", [[1, 2, 0], [0, 0, 0]])
@pytest.mark.parametrize("heads, max_new", [(2, 50), (8, 50), (8, 800)])
def test_max_new_is_only_a_bound(gp, heads, max_new, news, cache):
    """blocks of rows that no sequence has any rows in, a batch without new tokens among them: nothing is written there, and the launch ends"""
    seqs = S.Sequences([1500, 2100, 40], news, 64, gen(19), tail=3, max_new=max_new)
    a = Attend(gp, "f16", cache, seqs, heads, 2, 64, True, 20)
    a.launch()
    a.check()
    for dt in DTS:
        b = Append(gp, dt, "e4m3" if cache == "e4m3" else dt, seqs, heads, 2, 64, 64, "halves", 21)
        b.launch()
        b.check()


# ---- log probabilities -----------------------------------------------------------------------------------------------------


class Logprobs:
    def __init__(self, gp, dt, x, tokens, top, scale=1.0, ld=None, offset=0):
        self.gp, self.dt, self.top, self.scale = gp, dt, top, scale
        rows, vocab = x.shape
        ld = vocab if ld is None else ld
        self.x, self.tokens = x, tokens
        room = torch.full((rows * ld + offset,), math.nan, dtype=S.TORCH[dt])  # what lies between the rows counts for nothing
        room[offset:].view(rows, ld)[:, :vocab] = x
        self.room, self.t = room.cuda(), tokens.cuda()
        self.out = {"logprob": torch.full((rows,), 7.0).cuda(), "entropy": torch.full((rows,), 7.0).cuda(),
                    "ids": torch.full((rows, max(1, top)), 7, dtype=torch.int32).cuda(), "values": torch.full((rows, max(1, top)), 7.0).cuda()}
        self.p = gp.TokenLogprobsParams(dtype=gp.DTYPE_BY_NAME[dt], rows=rows, vocab=vocab, logits=self.room.data_ptr() + offset * self.room.element_size(), ld=ld, tokens=self.t.data_ptr(),
                                        scale=scale, logprob=self.out["logprob"].data_ptr(), entropy=self.out["entropy"].data_ptr(), top=top,
                                        top_ids=self.out["ids"].data_ptr(), top_logprobs=self.out["values"].data_ptr())
        n = gp.C.c_size_t()
        gp.check(gp.lib().gp_token_logprobs_work_bytes(gp.C.byref(self.p), gp.C.byref(n)))
        self.work = torch.zeros(max(16, n.value), dtype=torch.uint8, device="cuda")
        self.p.work, self.p.work_bytes = self.work.data_ptr() if n.value else None, n.value

    def launch(self, ctx=None, stream=None):
        return self.gp.launch("gp_launch_token_logprobs", self.p, ctx, stream)

    def left(self):
        torch.cuda.synchronize()
        return {n: x.cpu() for n, x in self.out.items()}

    def check(self):
        got = self.left()
        said, entropy, ids, values = S.logprobs(self.x, self.tokens, self.scale or 1.0, self.top)
        vocab = self.x.shape[1]
        # a thread adds up to vocab / 256 exponentials in turn, and their sums are added; an exponent and a difference are off by two units of fp32 each
        total = (vocab / 256 + 32) * 2.0 ** -24 + 2.0 ** -21

        def near(x, ref, what):
            assert torch.equal(x.isnan(), ref.isnan()), what
            assert torch.equal(x == -math.inf, ref == -math.inf), what
            fine = torch.isfinite(ref)
            assert ((x.double() - ref).abs() <= total + ref.abs() * 2.0 ** -21)[fine].all(), what

        near(got["logprob"], said, "logprob")
        fine = torch.isfinite(entropy)
        assert torch.equal(got["entropy"].isnan(), entropy.isnan())
        # every term p log p is off by a few units of its own, and by the error of the sum
        assert ((got["entropy"].double() - entropy).abs() <= 2 * total * (1 + entropy.abs()) + 2.0 ** -20)[fine].all()
        if self.top:
            assert torch.equal(got["ids"], ids)
            near(got["values"], values, "values")
        else:
            assert (got["ids"] == 7).all()


LOGPROBS = [
    # rows, vocab, top, scale, ld, offset
    (1, 1, 1, 1.0, None, 0),
    (3, 7, 32, 0.0, None, 0),  # fewer tokens than alternatives are asked for
    (5, 255, 5, 0.7, 259, 1),
    (2, 1000, 0, 1.0, None, 0),
    (4, 4099, 20, 2.0, None, 3),
    (1, 30522, 5, 1.0, None, 0),
    (3, 65537, 32, 1.0, 65600, 0),
    (600, 300, 3, 1.0, None, 0),
    (2, 8, 3, 1.0, None, 0), (2, 9, 4, 1.0, 16, 1), (1, 16384, 6, 1.0, None, 0), (2, 16385, 32, 1.0, None, 1),  # around a chunk, and around a tile
    (2, 131072 + 8, 20, 1.0, None, 0),  # in parts
]


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("case", range(len(LOGPROBS)))
def test_logprobs_match_their_definition(gp, dt, case):
    rows, vocab, top, scale, ld, offset = LOGPROBS[case]
    rng = gen(case)
    x = (3 * torch.randn((rows, vocab), generator=rng)).to(S.TORCH[dt])
    x[:, torch.rand(vocab, generator=rng) < 0.05] = -math.inf
    tokens = torch.randint(0, vocab, (rows,), generator=rng)
    if rows > 2:
        tokens[-1], tokens[-2] = -1, vocab  # padding
    a = Logprobs(gp, dt, x, tokens, top, scale, ld, offset)
    a.launch()
    a.check()
    first = a.left()
    a.launch()
    assert all(torch.equal(v, first[n]) for n, v in a.left().items())


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [100, 9001, 40000, 70000])
def test_logprobs_of_rows_of_a_kind(gp, dt, vocab):
    """rows that are masked all over, or but for a few, or with the type's lowest value; equal, rising and falling ones; zeros of both signs; NaN and infinity"""
    low = torch.finfo(S.TORCH[dt]).min
    x = torch.full((11, vocab), -math.inf)
    x[1, [3, vocab - 1, 50]] = torch.tensor([1.0, 2.0, 1.0])
    x[2] = low
    x[3] = low
    x[3, 77] = 5.0
    x[4] = 0.25
    x[5] = torch.arange(vocab) / 64.0
    x[6] = -torch.arange(vocab) / 64.0
    x[7], x[7, 1::2] = 0.0, -0.0
    x[8] = torch.randn(vocab, generator=gen(1))
    x[8, 9] = math.nan
    x[9] = torch.randn(vocab, generator=gen(2))
    x[9, 11] = math.inf
    x[10] = low
    x[10, 5] = -low
    x = x.to(S.TORCH[dt])
    tokens = torch.tensor([0, 3, 5, 77, 9, vocab - 1, 0, 1, 3, 12, 5])
    for scale in (1.0, 3.0):
        a = Logprobs(gp, dt, x, tokens, 20, scale)
        a.launch()
        got = a.left()
        fine = [r for r in range(11) if r not in (8, 9, 10) and not (scale > 1 and r in (2, 3))]
        a.x, a.tokens = x[fine], tokens[fine]
        a.out = {n: v[fine] for n, v in a.out.items()}
        a.check()
        for r in (8, 9):
            assert got["logprob"][r].isnan() and got["entropy"][r].isnan() and got["values"][r].isnan().all()
        assert 9 not in got["ids"][8] and got["ids"][9, 0] == 11 and (got["ids"][8:10] >= 0).all()
        # the largest value next to the lowest: one takes everything; the lowest everywhere: all are alike
        assert got["logprob"][10] == 0 and got["entropy"][10] == 0 and got["ids"][10, :2].tolist() == [5, 0] and got["logprob"][3] == 0
        assert abs(float(got["logprob"][2]) + math.log(vocab)) < 1e-5 * math.log(vocab) and got["ids"][2].tolist() == list(range(20))


def test_logprobs_of_more_tiles_than_are_kept_apart(gp):
    """as many rows as there are compute units, 33 tiles each: the first and the last share their groups' largest logits"""
    vocab = 32 * 16384 + 77
    x = torch.randn((256, vocab), generator=torch.Generator(device="cuda").manual_seed(5), device="cuda", dtype=torch.half)
    x[3, 5], x[3, vocab - 3], x[7, 16384 * 32 + 1] = 9.0, 9.0, 8.0
    tokens = torch.arange(256) * 2000
    out = {n: torch.empty(256, device="cuda") for n in ("logprob", "entropy")}
    ids, values = torch.empty((256, 12), dtype=torch.int32, device="cuda"), torch.empty((256, 12), device="cuda")
    t = tokens.cuda()
    p = gp.TokenLogprobsParams(dtype=gp.F16, rows=256, vocab=vocab, logits=x.data_ptr(), ld=vocab, tokens=t.data_ptr(), scale=1.0, logprob=out["logprob"].data_ptr(),
                               entropy=out["entropy"].data_ptr(), top=12, top_ids=ids.data_ptr(), top_logprobs=values.data_ptr())
    assert gp.launch("gp_launch_token_logprobs", p).total_tiles == 256
    torch.cuda.synchronize()
    for r in (0, 3, 7, 255):
        lp = torch.log_softmax(x[r].double(), 0)
        order = torch.sort(x[r].double(), descending=True, stable=True).indices[:12]
        assert torch.equal(ids[r].long(), order)
        # a thread adds 1056 exponentials in turn, of fp32's half unit each
        near = 1100 * 2.0 ** -24 + 16 * 2.0 ** -21
        assert (values[r].double() - lp[order]).abs().max() < near and abs(float(out["logprob"][r]) - float(lp[tokens[r]])) < near
        assert abs(float(out["entropy"][r]) + float((lp.exp() * lp).sum())) < 2 * near * 14


# ---- the forms that a call's size chooses -----------------------------------------------------------------------------------

MANY = [
    # lens, news, page, heads, kv_heads, dim, causal: blocks of 128 rows, which take 64 of them or more (heads x sequences x blocks)
    ([1300, 1100, 900, 70], [70, 66, 80, 70], 16, 16, 16, 64, True),       # keys in two parts; a sequence of nothing but its new tokens
    ([1300, 0, 64, 650], [70, 3, 0, 129], 64, 16, 16, 64, False),          # no keys, no rows, two blocks of rows
    ([700, 130, 65, 1], [50, 130, 2, 1], 128, 48, 16, 128, True),          # three query heads to a head: tokens that straddle blocks
    ([40, 300], [67, 65], 32, 32, 32, 128, True),                          # the first has tokens in front of position 0
]


@pytest.mark.parametrize("cache", ["same", "e4m3"])
@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("case", range(len(MANY)))
def test_attention_of_many_rows(gp, dt, cache, case):
    lens, news, page, heads, kv_heads, dim, causal = MANY[case]
    seqs = S.Sequences(lens, news, page, gen(40 + case), tail=1)
    a = Attend(gp, dt, dt if cache == "same" else cache, seqs, heads, kv_heads, dim, causal, 300 + case, scale=-0.3 if case == 2 else None, pad=8 * (case % 2))
    info = a.launch()
    assert info.block == 256 and info.total_tiles % (kv_heads * len(lens) * -(-seqs.max_new * heads // kv_heads // 128)) == 0
    a.check()
    first = a.left()
    a.launch()
    assert torch.equal(a.left(), first)


def test_attention_of_many_rows_and_keys(gp):
    """more heads than parts would help: every block walks over all keys, more than sixteen tiles of them; pages that are not there among them"""
    holes = {(0, 5): -1, (0, 16): 10 ** 6, (2, 0): -1}
    seqs = S.Sequences([1200, 3, 70, 0, 1, 2, 30, 9], [67, 1, 3, 0, 1, 2, 0, 1], 64, gen(50), holes=holes)
    a = Attend(gp, "bf16", "e4m3", seqs, 64, 64, 64, True, 51)
    a.launch()
    a.check()


def test_attention_of_more_sequences_than_a_wavefront_has_lanes(gp):
    """keys in equal parts over 70 sequences, one long and the others short, some of them empty"""
    lens = [1300] + [i * 37 % 41 for i in range(69)]
    for news in (None, [2] + [i % 3 for i in range(69)]):
        seqs = S.Sequences(lens, news, 16, gen(52))
        a = Attend(gp, "f16", "e4m3", seqs, 2, 1, 64, True, 53)
        a.launch()
        a.check()
        first = a.left()
        a.launch()
        assert torch.equal(a.left(), first)


def test_attention_of_a_part_longer_than_a_wavefronts_pages(gp):
    """256 heads: one part each, of more keys than 64 tiles for each wavefront"""
    seqs = S.Sequences([4400], None, 128, gen(54))
    a = Attend(gp, "f16", "e4m3", seqs, 256, 256, 64, True, 55)
    info = a.launch()
    assert info.total_tiles == 256
    a.check()


# ---- stopped and resumed, other streams, graphs -------------------------------------------------------------------------------


def calls(gp):
    """(a call, its outputs as bytes) of every kernel, with several tiles each"""
    out = []
    for cache, news in (("f16", None), ("e4m3", [100, 60, 33])):
        seqs = S.Sequences([200, 160, 133], news, 16, gen(60))
        out.append(Append(gp, "f16", cache, seqs, 4, 4, 64, 64, "halves", 61))
    out.append(Attend(gp, "f16", "f16", S.Sequences([2000, 700, 1], None, 64, gen(62)), 8, 4, 64, True, 63))
    out.append(Attend(gp, "bf16", "e4m3", S.Sequences([900, 300, 1500], [3, 1, 4], 32, gen(64)), 8, 4, 128, True, 65))
    out.append(Attend(gp, "bf16", "e4m3", S.Sequences([1300, 1100, 900, 70], [70, 66, 80, 70], 64, gen(66)), 16, 16, 64, True, 67))
    x = torch.randn((3, 70000), generator=gen(68)).half()
    out.append(Logprobs(gp, "f16", x, torch.tensor([1, 2, 3]), 20))
    out.append(Logprobs(gp, "f16", torch.randn((40, 900), generator=gen(69)).half(), torch.arange(40), 5))
    return out


def bits(left):
    return [x.contiguous().view(torch.uint8) for x in (left.values() if isinstance(left, dict) else [left])]


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(bits(a), bits(b)))


def clean(call):
    """What the call writes, as before its first launch"""
    if isinstance(call, Append):
        for n, x in call.cache.items():
            call.dev[n].copy_(x)
        call.q_out.fill_(7.0)
    elif isinstance(call, Attend):
        call.out.fill_(7.0)
    else:
        for x in call.out.values():
            x.fill_(7)
    torch.cuda.synchronize()


@pytest.mark.parametrize("which", range(7))
def test_stopped_and_resumed_has_the_bits_of_an_uninterrupted_launch(gp, which):
    call = calls(gp)[which]
    call.launch()
    want = call.left()
    for groups in (1, 32):
        flag = gp.Flag()
        st = gp.BlpState(1, flag, groups)
        clean(call)
        # (one counter: two workgroups, the second claim raises the flag; many: a bit or a count per workgroup)
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
    # ... and the next launch finds its workspace as it needs it
    clean(call)
    call.launch()
    assert same(call.left(), want)


def test_two_streams_at_once(gp):
    """each call with another of its kind on another stream, each with its own workspace and outputs"""
    first, second = calls(gp), calls(gp)
    want = []
    for c in first:
        c.launch()
        want.append(c.left())
        clean(c)
    streams = [gp.Stream(0), gp.Stream(1)]
    for _ in range(3):
        for a, b in zip(first, second):
            a.launch(stream=streams[0])
            b.launch(stream=streams[1])
        for s in streams:
            s.sync()
        for a, b, w in zip(first, second, want):
            assert same(a.left(), w) and same(b.left(), w)
            clean(a)
            clean(b)
    for s in streams:
        s.destroy()


def test_one_workspace_for_launches_of_any_sizes(gp):
    """as a program keeps it: of the largest size, zeroed once, for steps of few and of many sequences, short prompts and rows of logits, one after the other"""
    calls = []
    for lens, news, heads, kv_heads, dim in (([1500], None, 2, 2, 64), ([1500, 1100, 2000] * 20, None, 8, 4, 64), ([1700, 900], [1, 90], 16, 8, 128), ([2600] * 8, [70] * 8, 16, 2, 64),
                                             ([900, 3500], [9, 8], 8, 4, 64), ([3500] * 5, None, 16, 16, 128)):
        seqs = S.Sequences(lens, news, 64, gen(30))
        calls.append(Attend(gp, "bf16", "bf16", seqs, heads, kv_heads, dim, True, 31 + len(calls)))
    for rows, vocab in ((1, 300000), (100, 70000), (2, 66000)):
        calls.append(Logprobs(gp, "bf16", torch.randn((rows, vocab), generator=gen(40 + rows)).bfloat16(), torch.arange(rows), 32))
    assert all(c.p.work_bytes for c in calls)
    room = max(c.p.work_bytes for c in calls)
    shared = torch.zeros(room, dtype=torch.uint8, device="cuda")
    for c in calls:
        c.p.work, c.p.work_bytes = shared.data_ptr(), room
    for order in (calls, calls[::-1], calls[::2] + calls[1::2]):
        for c in order:
            c.launch()
        for c in order:
            c.check()
            for x in c.out.values() if isinstance(c, Logprobs) else [c.out]:
                x.fill_(7)


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("news", [None, [70, 40]])
def test_pages_and_rows_behind_four_gigabytes(gp, news, cache):
    """the last pages of a large pool, and rows far apart: the bits of the same call in a small one"""
    seqs = S.Sequences([700, 1300], news, 64, gen(80))
    app, att = Append(gp, "bf16", cache, seqs, 8, 4, 128, 128, "halves", 81), Attend(gp, "bf16", cache, seqs, 8, 4, 128, True, 82)
    att.p.cache = app.p.cache  # (one cache for both)
    att.p.q, att.p.ld_q = app.q_out.data_ptr(), app.q_out.shape[1]
    app.launch()
    att.launch()
    small = app.left(), att.left()
    clean(app)
    clean(att)
    block = 4 * 64 * 128 * app.dev["k"].element_size()
    pages = (5 << 30) // block
    big = {n: torch.empty((pages,) + tuple(app.dev[n].shape[1:]), dtype=app.dev[n].dtype, device="cuda") for n in app.cache}
    for n, x in app.cache.items():
        big[n][-seqs.pages:].copy_(x)
        setattr(app.p.cache, n, big[n].data_ptr())
    app.p.cache.pages = pages
    table = app.dev["table"] + (pages - seqs.pages)
    app.p.page_table = att.p.page_table = table.data_ptr()
    att.p.cache = app.p.cache
    ld = (1 << 32) // (seqs.tokens - 1) // 8 * 8 + 8  # the last row begins behind 2^32 values
    far_q, far_out = (torch.empty(ld * (seqs.tokens - 1) + 8 * 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    app.p.q_out, app.p.ld_q_out, att.p.q, att.p.ld_q, att.p.out, att.p.ld_out = far_q.data_ptr(), ld, far_q.data_ptr(), ld, far_out.data_ptr(), ld
    app.launch()
    att.launch()
    torch.cuda.synchronize()
    for n in app.cache:
        assert torch.equal(big[n][-seqs.pages:].cpu().view(torch.uint8), small[0][n].view(torch.uint8)), n
    for row in range(seqs.tokens):
        assert torch.equal(far_q[row * ld:row * ld + 1024].cpu(), small[0]["q"][row, :1024])
        assert torch.equal(far_out[row * ld:row * ld + 1024].cpu(), small[1][row, :1024])


def test_logits_behind_four_gigabytes(gp):
    x = (3 * torch.randn((5, 20000), generator=gen(83))).bfloat16()
    a = Logprobs(gp, "bf16", x, torch.arange(5), 10)
    ld = (1 << 30) + 1  # the last row begins behind 2^32 values
    far = torch.empty(4 * ld + 20000, dtype=torch.bfloat16, device="cuda")
    for row in range(5):
        far[row * ld:row * ld + 20000].copy_(x[row])
    a.p.logits, a.p.ld = far.data_ptr(), ld
    a.launch()
    a.check()


def test_captured_and_replayed(gp):
    """a step in a graph: replays with the program's own work in between, with other contents of the same buffers (lengths among them) every time"""
    stream = gp.Stream(0)
    news = None
    seqs = S.Sequences([1800, 900, 300], news, 32, gen(70))
    app, att = Append(gp, "bf16", "e4m3", seqs, 8, 4, 64, 64, "halves", 71), Attend(gp, "bf16", "e4m3", seqs, 8, 4, 64, True, 72)
    lp = Logprobs(gp, "f32", torch.randn((2, 70000), generator=gen(73)), torch.tensor([5, 6]), 7)
    for c in (app, att, lp):  # (what a first launch sets up is not part of the graph)
        c.launch(stream=stream)
    stream.sync()
    graph = gp.vp()
    gp.check(gp.lib().gp_graph_begin(stream.h))
    for c in (app, att, lp):
        c.launch(stream=stream)
    gp.check(gp.lib().gp_graph_end(stream.h, gp.C.byref(graph)))
    for i in range(4):
        lens = [1800 - 311 * i, 900 - i, 300 + 200 * i]
        for c in (app, att):
            c.dev["kv_len"].copy_(torch.tensor(lens, dtype=torch.int32))
        att.dev["q"].copy_(torch.randn(att.q.shape, generator=gen(80 + i)).bfloat16())
        lp.room.copy_(torch.randn(lp.room.shape, generator=gen(90 + i)))
        for name in ("k", "v", "k_scale", "v_scale"):  # (the second length is past what was filled: plain values)
            app.dev[name].copy_(app.cache[name].nan_to_num(0.5) if name in ("k_scale", "v_scale") else app.cache[name])
            att.dev[name].copy_(att.cache[name])
        for c in (app, att, lp):
            clean(c) if c is not app else app.q_out.fill_(7.0)
        torch.cuda.synchronize()
        before = {n: app.dev[n].clone() for n in app.cache}
        gp.check(gp.lib().gp_graph_launch(graph, stream.h))
        stream.sync()
        got = [app.left(), att.left(), lp.left()]
        for n, x in before.items():
            app.dev[n].copy_(x)
        for c in (app, att, lp):
            c.launch()
        for g, c in zip(got, (app, att, lp)):
            assert same(g, c.left()), (i, type(c))
    gp.check(gp.lib().gp_graph_destroy(graph))
    stream.destroy()


# ---- together -------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("cache", ["f16", "e4m3"])
def test_a_decoder_steps(gp, cache):
    """Two prompts, then eight steps of one token: every step appends, attends to what the cache then holds, projects (gp_launch_gemm) and scores, on
    one stream without a wait in between; each step's attention and scores against 64 bits, from the cache as it is."""
    heads, kv_heads, dim, page, vocab = 4, 2, 64, 16, 1000
    rng = gen(100)
    stream = gp.Stream(0)
    lens, news, steps = [37, 5], [37, 5], 8
    W = (0.05 * torch.randn((vocab, heads * dim), generator=rng)).half().cuda()
    seqs = S.Sequences([n + steps for n in lens], None, page, gen(101))
    pool = S.cache_of(seqs, kv_heads, dim, cache, rng)  # (its values are old ones: nothing of them may show)
    dev = {n: x.cuda() for n, x in pool.items()}
    inv_freq = 10000.0 ** (-torch.arange(0, dim, 2) / dim)
    freq = inv_freq.float().cuda()
    keep = []
    checks = []
    for step in range(steps + 1):
        if step:
            lens, news = [n + 1 for n in lens], [1, 1]
        s = S.Sequences(lens, None if step else news, page, gen(101), width=seqs.width)
        s.table, s.pages = seqs.table, seqs.pages
        d = {**s.device(), **dev}
        qkv = torch.randn((s.tokens, (heads + 2 * kv_heads) * dim), generator=rng).half().cuda()
        q, out = (torch.empty((s.tokens, heads * dim), dtype=torch.half, device="cuda") for _ in range(2))
        logits = torch.empty((s.tokens, vocab), dtype=torch.half, device="cuda")
        tokens = torch.randint(0, vocab, (s.tokens,), generator=rng).cuda()
        lp = {n: torch.empty(s.tokens, device="cuda") for n in ("logprob", "entropy")}
        ids, vals = torch.empty((s.tokens, 4), dtype=torch.int32, device="cuda"), torch.empty((s.tokens, 4), device="cuda")
        c = S.cache_params(gp, d, cache, kv_heads, dim, s)
        at, es = qkv.data_ptr(), 2 * dim
        torch.cuda.synchronize()  # (the inputs were made on torch's stream)
        gp.launch("gp_launch_kv_append", gp.KvAppendParams(dtype=gp.F16, cache=c, **S.sequence_params(s, d), heads=heads, q=at, k=at + es * heads, v=at + es * (heads + kv_heads),
                                                           ld_qkv=qkv.shape[1], q_out=q.data_ptr(), ld_q_out=heads * dim, inv_freq=freq.data_ptr(), rot_dim=dim, rot_pairs=gp.ROT_HALVES), stream=stream)
        gp.launch("gp_launch_paged_attention", gp.PagedAttentionParams(dtype=gp.F16, cache=c, **S.sequence_params(s, d), heads=heads, max_len=64, q=q.data_ptr(), ld_q=heads * dim,
                                                                       out=out.data_ptr(), ld_out=heads * dim, scale=0.125, causal=1), stream=stream)
        gp.launch("gp_launch_gemm", gp.GemmParams(dtype=gp.F16, M=s.tokens, N=vocab, K=heads * dim, A=out.data_ptr(), lda=heads * dim, B=W.data_ptr(), ldb=heads * dim, b_is_nk=1,
                                                  C=logits.data_ptr(), ldc=vocab, alpha=1.0, batch=1), stream=stream)
        gp.launch("gp_launch_token_logprobs", gp.TokenLogprobsParams(dtype=gp.F16, rows=s.tokens, vocab=vocab, logits=logits.data_ptr(), ld=vocab, tokens=tokens.data_ptr(), scale=1.0,
                                                                     logprob=lp["logprob"].data_ptr(), entropy=lp["entropy"].data_ptr(), top=4, top_ids=ids.data_ptr(), top_logprobs=vals.data_ptr()), stream=stream)
        keep.append((d, qkv, tokens))
        stream.sync()
        now = {n: x.cpu() for n, x in dev.items()}
        # the keys that this step appended, rotated in 64 bits, are in the cache up to its rounding
        for b in range(2):
            for row, pos in s.rows(b):
                page_, slot = s.place(b, pos)
                ref = S.turned(qkv[row, heads * dim: (heads + kv_heads) * dim].cpu().double().view(kv_heads, dim), pos, inv_freq.float(), dim, "halves")
                assert ((S.values(now, "k")[page_, :, slot] - ref).abs() <= (2.0 ** -11 if cache == "f16" else 2.0 ** -4) * ref.abs() + (2e-5 if cache == "f16" else 2.0 ** -6)).all()
        want, mass, most = S.attend(s, now, q.cpu().view(s.tokens, heads, dim), 0.125, True)
        for row, ref in want.items():
            # (as for the attention alone: two roundings to fp16, a score's products and sums in fp32)
            allowed = 2.0 ** -11 * (mass[row] + ref.abs()) + 4 * (dim + 8) * 2.0 ** -24 * max(most, 1.0) * mass[row] + 2.0 ** -24 * (1 + 64 * mass[row].amax())
            assert ((out[row].cpu().view(heads, dim).double() - ref).abs() <= allowed).all()
        said, entropy, wids, wvals = S.logprobs(logits.cpu(), tokens.cpu(), 1.0, 4)
        assert (lp["logprob"].cpu().double() - said).abs().max() < 4e-6 and (lp["entropy"].cpu().double() - entropy).abs().max() < 2e-5
        assert torch.equal(ids.cpu(), wids) and (vals.cpu().double() - wvals).abs().max() < 4e-6
    stream.destroy()
