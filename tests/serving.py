"""A decoder's serving step in 64 bits, from the definitions in include/gpreempt_hip.h, and what the tests need to call the kernels."""
import math

import torch

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
LOWEST = 2.0 ** -40


def half_step(dt):
    """half a unit of the type, relative"""
    return torch.finfo(TORCH[dt]).eps / 2


class Sequences:
    """lens: tokens in the cache of each sequence, the new ones included; news: new tokens (None: one each, without a start array);
    holes: (sequence, entry) -> page number that is written into the table instead"""

    def __init__(self, lens, news, page, rng, spare=2, width=None, holes=None, tail=0, max_new=None):
        self.lens, self.page, self.batch = list(lens), page, len(lens)
        self.news = [1] * self.batch if news is None else list(news)
        self.start = None if news is None else [sum(self.news[:i]) for i in range(self.batch + 1)]
        self.tokens = sum(self.news) + tail  # rows behind the last sequence
        self.width = max(1, max(-(-n // page) for n in self.lens)) if width is None else width
        self.pages = self.batch * self.width + spare
        order = torch.randperm(self.pages, generator=rng)[: self.batch * self.width].reshape(self.batch, self.width).to(torch.int32)
        for at, number in (holes or {}).items():
            order[at] = number
        self.table = order
        self.max_new = max(1, max(self.news)) if max_new is None else max_new

    def rows(self, b):
        """(row, position) of sequence b's new tokens that a call handles"""
        r0 = b if self.start is None else self.start[b]
        n = self.news[b]
        return [(r0 + i, self.lens[b] - n + i) for i in range(min(n, self.max_new))]

    def place(self, b, pos):
        """(page, slot) of a position, or None"""
        if pos < 0 or pos // self.page >= self.width:
            return None
        page = int(self.table[b, pos // self.page])
        return (page, pos % self.page) if 0 <= page < self.pages else None

    def device(self):
        dev = {"kv_len": torch.tensor(self.lens, dtype=torch.int32).cuda(), "table": self.table.contiguous().cuda()}
        dev["start"] = None if self.start is None else torch.tensor(self.start, dtype=torch.int32).cuda()
        return dev


def cache_of(seqs, kv_heads, dim, cache, rng, size=1.0, poison=True):
    """A pool with random values where the sequences' older and newer tokens are and, with `poison`, NaN everywhere else:
    {"k", "v"} in the cache's type on the CPU, {"k_scale", "v_scale"} in fp32 for e4m3"""
    got = {}
    used = torch.zeros((seqs.pages, seqs.page), dtype=torch.bool)
    for b in range(seqs.batch):
        for pos in range(max(0, seqs.lens[b])):
            at = seqs.place(b, pos)
            if at:
                used[at] = True
    for name in ("k", "v"):
        x = size * torch.randn((seqs.pages, kv_heads, seqs.page, dim), generator=rng)
        if cache == "e4m3":
            scale = 2.0 ** torch.randint(-8, 3, (seqs.pages, kv_heads), generator=rng).float() * (1 + torch.rand((seqs.pages, kv_heads), generator=rng))
            got[name + "_scale"] = scale
            x = x * 20.0 / size  # (e4m3 has its full precision from 2^-6 on)
        x = x.to(TORCH[cache])
        if poison:
            bits = x.view(torch.uint8 if cache == "e4m3" else torch.int16)
            bits[~used[:, None, :, None].expand_as(bits)] = 0x7F if cache == "e4m3" else 0x7FFF
        got[name] = x
    return got


def values(cache, name):
    x = cache[name].double()
    return x * cache[name + "_scale"].double()[:, :, None, None] if name + "_scale" in cache else x


def cache_params(gp, dev, cache_dtype, kv_heads, dim, seqs):
    e8 = cache_dtype == "e4m3"
    return gp.KvCache(dtype=gp.E4M3 if e8 else gp.DTYPE_BY_NAME[cache_dtype], kv_heads=kv_heads, head_dim=dim, page_size=seqs.page, pages=seqs.pages, k=dev["k"].data_ptr(),
                      v=dev["v"].data_ptr(), k_scale=dev["k_scale"].data_ptr() if e8 else None, v_scale=dev["v_scale"].data_ptr() if e8 else None)


def sequence_params(seqs, dev):
    return dict(batch=seqs.batch, tokens=seqs.tokens, max_new=seqs.max_new, start=None if dev["start"] is None else dev["start"].data_ptr(), kv_len=dev["kv_len"].data_ptr(),
                page_table=dev["table"].data_ptr(), table_width=seqs.width)


def turned(x, pos, inv_freq, rot, pairs):
    """heads x dim in 64 bits"""
    y = x.clone()
    for j in range(rot // 2):
        i0, i1 = (j, j + rot // 2) if pairs == "halves" else (2 * j, 2 * j + 1)
        angle = pos * float(inv_freq[j])
        c, s = math.cos(angle), math.sin(angle)
        y[..., i0], y[..., i1] = x[..., i0] * c - x[..., i1] * s, x[..., i1] * c + x[..., i0] * s
    return y


def scale_for(most):
    if most == 0:
        return LOWEST
    k = math.ceil(math.log2(most / 448))
    k += most > 448 * 2.0 ** k
    k -= most <= 448 * 2.0 ** (k - 1)
    return max(LOWEST, 2.0 ** k)


def append(seqs, cache, cache_dtype, k, v, rot, pairs, inv_freq):
    """The cache after an append, in 64 bits and (8 bits) before the rounding to e4m3: ({"k", "v"}, scales, written slots [page, slot],
    entries (name, page, head) whose other slots were put on a new scale)"""
    new = {n: cache[n].double().clone() for n in ("k", "v")}
    scales = {n: cache[n + "_scale"].double().clone() for n in ("k", "v")} if cache_dtype == "e4m3" else None
    written, again = torch.zeros((seqs.pages, seqs.page), dtype=torch.bool), set()
    by_page, first = {}, set()
    for b in range(seqs.batch):
        for row, pos in seqs.rows(b):
            at = seqs.place(b, pos)
            if at:
                if pos // seqs.page == max(0, seqs.rows(b)[0][1]) // seqs.page:
                    first.add(at[0])
                written[at] = True
                by_page.setdefault(at[0], []).append((at[1], row, pos))
    for page, rows in by_page.items():
        for name, src in (("k", k), ("v", v)):
            x = {slot: turned(src[row].double(), pos, inv_freq, rot if name == "k" else 0, pairs) for slot, row, pos in rows}
            if scales is None:
                for slot, y in x.items():
                    new[name][page, :, slot] = y
                continue
            for h in range(new[name].shape[1]):
                finite = torch.cat([y[h][torch.isfinite(y[h])] for y in x.values()])
                most = float(finite.abs().max()) if finite.numel() else 0.0
                before = 0.0 if 0 in x else float(scales[name][page, h])
                scale = before if 0 < before < math.inf and most <= 448 * before else scale_for(most)
                if scale != before and page in first:
                    new[name][page, h] *= (before if 0 < before < math.inf else 0.0) / scale
                    again.add((name, page, h))
                scales[name][page, h] = scale
                for slot, y in x.items():
                    new[name][page, h, slot] = (y[h] / scale).clamp(-448, 448)
    return new, scales, written, again


def attend(seqs, cache, q, scale, causal, max_len=None):
    """tokens x heads x dim in 64 bits, None for rows that no call writes; and sum_j p_j |v_j|, and sum_j |q k| scale at its largest"""
    K, V = values(cache, "k"), values(cache, "v")
    heads, dim, kv_heads = q.shape[1], q.shape[2], K.shape[1]
    out, mass, most = {}, {}, 0.0
    for b in range(seqs.batch):
        places = [seqs.place(b, p) for p in range(max(0, seqs.lens[b] if max_len is None else min(seqs.lens[b], max_len)))]
        for row, pos in seqs.rows(b):
            at = [a for p, a in enumerate(places) if a and (not causal or p <= pos)]
            o, m = torch.zeros(heads, dim, dtype=torch.float64), torch.zeros(heads, dim, dtype=torch.float64)
            if at:
                pages, slots = torch.tensor(at).t()
                k, v = K[pages, :, slots], V[pages, :, slots]  # keys x kv_heads x dim
                for h in range(heads):
                    x, g = q[row, h].double(), h // (heads // kv_heads)
                    p = torch.softmax(k[:, g] @ x * scale, 0)
                    o[h], m[h] = p @ v[:, g], p @ v[:, g].abs()
                    most = max(most, float((k[:, g].abs() @ x.abs()).max()) * abs(scale))
            out[row], mass[row] = o, m
    return out, mass, most


def logprobs(x, tokens, scale, top):
    """in 64 bits: (logprob, entropy, ids, values); x: rows x vocab"""
    y = x.double() * scale
    empty = (x == -math.inf).all(-1)
    lp = torch.log_softmax(y, -1)
    p = lp.exp()
    entropy = torch.where(p > 0, -p * lp, torch.where(p.isnan(), p, 0.0)).sum(-1)
    entropy[empty] = 0.0
    said = torch.zeros(len(x), dtype=torch.float64)
    ids, vals = torch.full((len(x), top), -1, dtype=torch.int32), torch.full((len(x), top), -math.inf, dtype=torch.float64)
    for r in range(len(x)):
        t = int(tokens[r])
        if 0 <= t < x.shape[1]:
            said[r] = -math.inf if empty[r] else lp[r, t]
        order = sorted((-float(v), i) for i, v in enumerate(x[r].double().tolist()) if v > -math.inf)[:top]
        for i, (_, at) in enumerate(order):
            ids[r, i], vals[r, i] = at, lp[r, at]
    return said, entropy, ids, vals
