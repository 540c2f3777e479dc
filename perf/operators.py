"""What a decoder's serving step needs next to the matrix products: new keys and values go into a paged cache with the
position rotation applied on the way, queries attend to what the cache holds, and the logits become log probabilities.

A case is a dict of plain values.  There are three kinds:

  append    gp_launch_kv_append: rows of packed q, k, v of some sequences; k and v go to the sequences' pages, in 16 bits or in
            8 bits with a scale for each page and head, and q is rotated into a tensor of its own.
  attend    gp_launch_paged_attention: the queries of the sequences' last tokens (or of a decoder's tokens over an encoder's
            states: not causal) over the pages.
  logprobs  gp_launch_token_logprobs: for each row of logits the log probability of a given token, the entropy and the
            largest alternatives.

Where `own` is false the operators are computed in elementary torch operations."""
import math
import random

import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1}
LOWEST_SCALE = 2.0 ** -40  # of a page in 8 bits


def listed():
    gqa = {"heads": 32, "kv_heads": 8, "head_dim": 128}  # four query heads to a head of the cache
    mha = {"heads": 12, "kv_heads": 12, "head_dim": 64}  # the head layout of the framework's BERT-base
    return [
        # the smallest call: one user's next token, 16-bit cache in small pages
        {"name": "append_one_bf16", "kind": "append", "dtype": "bf16", "cache": "bf16", **mha, "page": 16, "batch": 1, "new": 1, "len": 211, "rot": 64, "pairs": "halves"},
        # a step of 64 users at once: most tokens land in pages that hold others already
        {"name": "append_step_b64_e4m3", "kind": "append", "dtype": "bf16", "cache": "e4m3", **gqa, "page": 64, "batch": 64, "new": 1, "len": 2048, "rot": 128, "pairs": "halves"},
        # ragged pieces of prompts behind what is there
        {"name": "append_prompts_e4m3", "kind": "append", "dtype": "f16", "cache": "e4m3", **gqa, "page": 64, "batch": 5, "new": 1777, "len": 2500, "rot": 128, "pairs": "halves"},
        # one long prompt, half of a head rotated, in neighbouring pairs
        {"name": "append_prompt_bf16", "kind": "append", "dtype": "bf16", "cache": "bf16", **gqa, "page": 32, "batch": 1, "new": 8192, "len": 8192, "rot": 64, "pairs": "neighbours"},
        # the smallest call: one user's next token
        {"name": "attend_one_f16", "kind": "attend", "dtype": "f16", "cache": "f16", **mha, "page": 16, "batch": 1, "new": 1, "len": 211, "causal": True},
        # a step of 64 users with contexts of all lengths, cache in 8 bits: the everyday load of a server
        {"name": "attend_step_b64_e4m3", "kind": "attend", "dtype": "bf16", "cache": "e4m3", **gqa, "page": 64, "batch": 64, "new": 1, "len": 8192, "causal": True},
        # one user with a very long context
        {"name": "attend_step_long_e4m3", "kind": "attend", "dtype": "f16", "cache": "e4m3", **gqa, "page": 64, "batch": 1, "new": 1, "len": 131072, "causal": True},
        # three guessed tokens and the next one of 24 users, 16-bit cache
        {"name": "attend_guesses_b24_bf16", "kind": "attend", "dtype": "bf16", "cache": "bf16", **gqa, "page": 32, "batch": 24, "new": 4, "len": 4001, "causal": True},
        # prompts of several users, cache in 8 bits: bound by the matrix products
        {"name": "attend_prompts_e4m3", "kind": "attend", "dtype": "bf16", "cache": "e4m3", **gqa, "page": 64, "batch": 4, "new": 4096, "len": 5000, "causal": True},
        # a decoder's tokens over an encoder's states: BERT-base's heads, the sequence length of the heaviest scenario
        {"name": "attend_encoder_f16", "kind": "attend", "dtype": "f16", "cache": "f16", **mha, "page": 64, "batch": 8, "new": 211, "len": 384, "causal": False},
        # one row over BERT's vocabulary: the next token of one user
        {"name": "logprobs_one_f32", "kind": "logprobs", "dtype": "f32", "rows": 1, "vocab": 30522, "top": 5},
        # a prompt scored token by token, with twenty alternatives each
        {"name": "logprobs_prompt_bf16", "kind": "logprobs", "dtype": "bf16", "rows": 500, "vocab": 131001, "top": 20},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "append", "attend", "attend", "attend", "logprobs"])
    if kind == "logprobs":
        vocab = _log(rng, 1000, 131072)
        return {"kind": kind, "dtype": rng.choice(["f32", "f16", "bf16"]), "rows": _log(rng, 1, max(1, min(500, 60_000_000 // vocab))), "vocab": vocab, "top": rng.randint(0, 20)}
    dtype, kv_heads, head_dim = rng.choice(["f16", "bf16"]), rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 128])
    case = {"kind": kind, "dtype": dtype, "cache": rng.choice([dtype, "e4m3", "e4m3"]), "heads": kv_heads * rng.choice([1, 2, 3, 4, 8]), "kv_heads": kv_heads,
            "head_dim": head_dim, "page": rng.choice([16, 32, 64, 128])}
    if rng.random() < 0.5:  # a step of many users
        batch, new = _log(rng, 1, 64), rng.choice([1, 1, 1, 2, 5])
        case.update(batch=batch, new=new, len=_log(rng, max(16, new), min(65536, 262144 // batch)))
    else:  # prompts
        new = _log(rng, 16, 4096)
        case.update(batch=_log(rng, 1, max(1, min(8, 8192 // new))), new=new, len=_log(rng, new, 5000))
    if kind == "append":
        case.update(len=min(case["len"], max(4096, case["new"])), rot=rng.choice([head_dim, head_dim, head_dim // 2, 0]), pairs=rng.choice(["halves", "neighbours"]))
    else:
        case.update(causal=rng.random() < 0.8)
    return case


def _lengths(case):
    """Tokens in the cache and new tokens of each sequence: the first has the largest numbers of the case."""
    rng = random.Random(case["batch"] * 1000003 + case["len"] * 1009 + case["new"])
    lens, news = [case["len"]], [case["new"]]
    for _ in range(case["batch"] - 1):
        n = case["new"] if case["new"] <= 8 else rng.randint(case["new"] // 4, case["new"])
        news.append(n)
        lens.append(rng.randint(max(n, case["len"] // 4), case["len"]))
    return lens, news


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _scale_of(most):
    """The smallest power of two that brings `most` to at most 448, the largest e4m3 value."""
    m, e = torch.frexp(most)
    return torch.where(most > 0, torch.ldexp(torch.ones_like(most), e - 9 + (m > 0.875).to(e.dtype)), 0.0).clamp_min(LOWEST_SCALE)


def _prepare_pages(case, gen):
    lens, news = _lengths(case)
    page, batch = case["page"], case["batch"]
    width = -(-case["len"] // page)
    pages = batch * width + 3
    shape = (pages, case["kv_heads"], page, case["head_dim"])
    st = {"case": case, "batch": batch, "tokens": sum(news), "width": width, "pages": pages, "max_new": max(news), "max_len": max(lens),
          "kv_len": _ints(lens), "start": None if case["new"] == 1 else _ints([sum(news[:i]) for i in range(batch + 1)]),
          # the pages of a sequence lie anywhere in the pool
          "table": torch.randperm(pages, generator=gen, device="cuda")[: batch * width].reshape(batch, width).to(torch.int32)}
    for name in ("k", "v"):
        x = torch.randn(shape, generator=gen, device="cuda", dtype=TORCH[case["dtype"]])
        # a head's keys and values have a size of their own
        x *= torch.rand((1, case["kv_heads"], 1, 1), generator=gen, device="cuda", dtype=x.dtype) + 0.5
        if case["cache"] == "e4m3":
            scale = _scale_of(x.abs().amax((2, 3)).float())
            st[name + "_scale"] = scale
            x = (x.float() / scale[:, :, None, None]).to(TORCH["e4m3"]).view(torch.uint8)
        st[name + "_cache"] = x
    return st


def _prepare_append(case, gen):
    st = _prepare_pages(case, gen)
    rows = (case["heads"] + 2 * case["kv_heads"]) * case["head_dim"]  # a row of the projection: q, k and v of one token
    st["qkv"] = torch.randn((st["tokens"], rows), generator=gen, device="cuda", dtype=TORCH[case["dtype"]])
    st["q_out"] = torch.empty((st["tokens"], case["heads"] * case["head_dim"]), device="cuda", dtype=TORCH[case["dtype"]])
    st["inv_freq"] = (10000.0 ** (-torch.arange(0, case["rot"], 2, dtype=torch.float64) / max(1, case["rot"]))).float().cuda()
    return st


def _prepare_attend(case, gen):
    st = _prepare_pages(case, gen)
    shape = (st["tokens"], case["heads"] * case["head_dim"])
    st["q"] = torch.randn(shape, generator=gen, device="cuda", dtype=TORCH[case["dtype"]])
    st["out"] = torch.empty_like(st["q"])
    return st


def _prepare_logprobs(case, gen):
    rows, vocab = case["rows"], case["vocab"]
    x = 2.5 * torch.randn((rows, vocab), generator=gen, device="cuda", dtype=TORCH[case["dtype"]])
    # what may not be said is masked: some tokens of the vocabulary in every row
    x[:, torch.rand((vocab,), generator=gen, device="cuda") < 0.01] = -math.inf
    tokens = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
    x[torch.arange(rows, device="cuda"), tokens] = 3.0  # a token that was said was not masked
    if rows > 4:
        tokens[-2:] = -1  # padding
    st = {"case": case, "logits": x, "tokens": tokens, "logprob": torch.empty(rows, device="cuda"), "entropy": torch.empty(rows, device="cuda")}
    if case["top"]:
        st["top_ids"] = torch.empty((rows, case["top"]), device="cuda", dtype=torch.int32)
        st["top_logprobs"] = torch.empty((rows, case["top"]), device="cuda")
    return st


PREPARE = {"append": _prepare_append, "attend": _prepare_attend, "logprobs": _prepare_logprobs}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return PREPARE[case["kind"]](case, gen)


# ---- the plain form --------------------------------------------------------------------------------------------------


def _sequences(st):
    """For each row of new tokens its sequence, and its position."""
    ids = torch.arange(st["batch"], device="cuda")
    if st["start"] is None:
        return ids, st["kv_len"].long() - 1
    start = st["start"].long()
    seq = torch.repeat_interleave(ids, start.diff(), output_size=st["tokens"])
    return seq, st["kv_len"].long()[seq] - start[seq + 1] + torch.arange(st["tokens"], device="cuda")


def _rotate(x, cos, sin, rot, pairs):
    """x: tokens x heads x head_dim in fp32; cos, sin: tokens x rot / 2"""
    cos, sin = cos[:, None], sin[:, None]
    if pairs == "halves":
        a, b = x[..., : rot // 2], x[..., rot // 2: rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([turned, x[..., rot:]], -1)


def _append_e4m3(cache, scale, x, st, page, slot):
    """x: tokens x kv_heads x head_dim in fp32.  A page's scale is set when its first token comes, and raised when a larger value does."""
    pages, kv_heads, size, dim = cache.shape
    most = torch.zeros((pages, kv_heads), device="cuda").index_reduce_(0, page, x.abs().amax(-1), "amax")
    fresh = torch.zeros(pages, dtype=torch.bool, device="cuda").index_fill_(0, page[slot == 0], True)
    before = torch.where(fresh[:, None], 0.0, scale)
    after = torch.where(most > 448 * before, _scale_of(most), before)
    after = torch.where(fresh[:, None], after.clamp_min(LOWEST_SCALE), after)
    # only the first page that a sequence writes to can hold older tokens
    n = torch.ones_like(st["kv_len"]) if st["start"] is None else st["start"].diff()
    first = st["table"].gather(1, ((st["kv_len"] - n) // size).long()[:, None])[:, 0].long()
    ratio = (before / after)[first]
    old = cache[first]
    again = (old.view(TORCH["e4m3"]).float() * ratio[:, :, None, None]).to(TORCH["e4m3"]).view(torch.uint8)
    cache[first] = torch.where((ratio == 1)[:, :, None, None], old, again)
    touched = torch.zeros(pages, dtype=torch.bool, device="cuda").index_fill_(0, page, True)
    scale.copy_(torch.where(touched[:, None], after, scale))
    cache[page, :, slot] = (x / scale[page][:, :, None]).clamp(-448, 448).to(TORCH["e4m3"]).view(torch.uint8)


def _plain_append(st):
    c = st["case"]
    dtype, heads, kv_heads, dim = TORCH[c["dtype"]], c["heads"], c["kv_heads"], c["head_dim"]
    seq, pos = _sequences(st)
    angle = pos.double()[:, None] * st["inv_freq"].double()
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    q, k, v = st["qkv"].float().view(-1, heads + 2 * kv_heads, dim).split([heads, kv_heads, kv_heads], 1)
    q, k = _rotate(q, cos, sin, c["rot"], c["pairs"]), _rotate(k, cos, sin, c["rot"], c["pairs"])
    st["q_out"].copy_(q.reshape(st["q_out"].shape))
    page, slot = st["table"][seq, pos // c["page"]].long(), pos % c["page"]
    if c["cache"] == "e4m3":
        _append_e4m3(st["k_cache"], st["k_scale"], k, st, page, slot)
        _append_e4m3(st["v_cache"], st["v_scale"], v, st, page, slot)
    else:
        st["k_cache"][page, :, slot] = k.to(dtype)
        st["v_cache"][page, :, slot] = v.to(dtype)


def _dense(st, name):
    """The pages of every sequence one behind the other, in fp32: batch x kv_heads x keys x head_dim"""
    table = st["table"].long()
    x = st[name + "_cache"]
    if st["case"]["cache"] == "e4m3":
        x = x[table].view(TORCH["e4m3"]).float() * st[name + "_scale"][table][..., None, None]
    else:
        x = x[table].float()
    return x.transpose(1, 2).flatten(2, 3)


def _plain_attend(st):
    c = st["case"]
    batch, kv_heads, dim, group, n = st["batch"], c["kv_heads"], c["head_dim"], c["heads"] // c["kv_heads"], st["max_new"]
    k, v = _dense(st, "k"), _dense(st, "v")
    start = torch.arange(batch + 1, device="cuda") if st["start"] is None else st["start"].long()
    count, step = start.diff(), torch.arange(n, device="cuda")
    row = (start[:-1, None] + step).clamp_max(st["tokens"] - 1)  # batch x n; those behind a sequence's last are not used
    q = st["q"].float().view(-1, kv_heads, group, dim)[row].permute(0, 2, 1, 3, 4).reshape(batch, kv_heads, n * group, dim)
    seen = st["kv_len"].long()[:, None] - (count[:, None] - 1 - step if c["causal"] else torch.zeros_like(step))  # keys that a query sees
    hidden = torch.arange(k.shape[2], device="cuda") >= seen.repeat_interleave(group, 1)[:, None, :, None]
    s = torch.matmul(q, k.transpose(2, 3)).mul_(dim ** -0.5).masked_fill_(hidden, -math.inf)
    s = torch.exp(s - s.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min))
    o = torch.matmul(s, v) / s.sum(-1, keepdim=True).clamp_min(1e-30)
    o = o.view(batch, kv_heads, n, group, dim).transpose(1, 2).reshape(batch, n, kv_heads * group * dim)
    seq = _sequences(st)[0]
    st["out"].copy_(o[seq, torch.arange(st["tokens"], device="cuda") - start[seq]])


def _plain_logprobs(st):
    x = st["logits"].float()
    y = x - x.amax(-1, keepdim=True)
    e = torch.exp(y)
    total = e.sum(-1)
    log_total = torch.log(total)
    st["entropy"].copy_(log_total - torch.where(e > 0, e * y, 0.0).sum(-1) / total)
    said = y.gather(1, st["tokens"].clamp_min(0)[:, None])[:, 0] - log_total
    st["logprob"].copy_(torch.where(st["tokens"] < 0, 0.0, said))
    if st["case"]["top"]:
        values, ids = torch.sort(y, dim=-1, descending=True, stable=True)
        st["top_ids"].copy_(ids[:, : st["case"]["top"]])
        st["top_logprobs"].copy_(values[:, : st["case"]["top"]] - log_total[:, None])


# ---- the framework's operators ------------------------------------------------------------------------------------------


def _cache_params(gp, st):
    c = st["case"]
    scales = [st[n].data_ptr() if c["cache"] == "e4m3" else None for n in ("k_scale", "v_scale")]
    return gp.KvCache(dtype=gp.E4M3 if c["cache"] == "e4m3" else gp.DTYPE_BY_NAME[c["cache"]], kv_heads=c["kv_heads"], head_dim=c["head_dim"], page_size=c["page"],
                      pages=st["pages"], k=st["k_cache"].data_ptr(), v=st["v_cache"].data_ptr(), k_scale=scales[0], v_scale=scales[1])


def _sequence_params(st):
    return {"batch": st["batch"], "tokens": st["tokens"], "max_new": st["max_new"], "start": None if st["start"] is None else st["start"].data_ptr(),
            "kv_len": st["kv_len"].data_ptr(), "page_table": st["table"].data_ptr(), "table_width": st["width"]}


def _append_params(gp, st):
    c = st["case"]
    at, size = st["qkv"].data_ptr(), st["qkv"].element_size() * c["head_dim"]
    return gp.KvAppendParams(dtype=gp.DTYPE_BY_NAME[c["dtype"]], cache=_cache_params(gp, st), **_sequence_params(st), heads=c["heads"],
                             q=at, k=at + size * c["heads"], v=at + size * (c["heads"] + c["kv_heads"]), ld_qkv=st["qkv"].shape[1],
                             q_out=st["q_out"].data_ptr(), ld_q_out=st["q_out"].shape[1], inv_freq=st["inv_freq"].data_ptr() if c["rot"] else None, rot_dim=c["rot"],
                             rot_pairs=gp.ROT_HALVES if c["pairs"] == "halves" else gp.ROT_NEIGHBOURS)


def _workspace(gp, st, p, entry):
    """What a program allocates once and keeps for its calls: zeroed before the first."""
    n = gp.C.c_size_t()
    gp.check(getattr(gp.lib(), entry)(gp.C.byref(p), gp.C.byref(n)))
    st["work"] = torch.zeros(max(1, n.value), dtype=torch.uint8, device="cuda")
    p.work, p.work_bytes = st["work"].data_ptr(), n.value


def _attend_params(gp, st):
    c = st["case"]
    p = gp.PagedAttentionParams(dtype=gp.DTYPE_BY_NAME[c["dtype"]], cache=_cache_params(gp, st), **_sequence_params(st), heads=c["heads"], max_len=st["max_len"],
                                q=st["q"].data_ptr(), ld_q=st["q"].shape[1], out=st["out"].data_ptr(), ld_out=st["out"].shape[1],
                                scale=c["head_dim"] ** -0.5, causal=int(c["causal"]))
    _workspace(gp, st, p, "gp_paged_attention_work_bytes")
    return p


def _logprobs_params(gp, st):
    c, top = st["case"], st["case"]["top"]
    p = gp.TokenLogprobsParams(dtype=gp.DTYPE_BY_NAME[c["dtype"]], rows=c["rows"], vocab=c["vocab"], logits=st["logits"].data_ptr(), ld=c["vocab"],
                               tokens=st["tokens"].data_ptr(), scale=1.0, logprob=st["logprob"].data_ptr(), entropy=st["entropy"].data_ptr(), top=top,
                               top_ids=st["top_ids"].data_ptr() if top else None, top_logprobs=st["top_logprobs"].data_ptr() if top else None)
    _workspace(gp, st, p, "gp_token_logprobs_work_bytes")
    return p


ENTRY = {"append": ("gp_launch_kv_append", _append_params), "attend": ("gp_launch_paged_attention", _attend_params), "logprobs": ("gp_launch_token_logprobs", _logprobs_params)}
PLAIN = {"append": _plain_append, "attend": _plain_attend, "logprobs": _plain_logprobs}


def run(state):
    kind = state["case"]["kind"]
    if own:
        from gpreempt_amd import capi as gp
        entry, params = ENTRY[kind]
        if "params" not in state:  # a program fills the struct in once and calls with it step after step
            gp.init(0)
            state["params"] = params(gp, state)
        gp.launch(entry, state["params"])
    else:
        PLAIN[kind](state)
    if kind == "attend":
        return state["out"]
    if kind == "logprobs":
        return {n: state[n] for n in ("logprob", "entropy", "top_ids", "top_logprobs") if n in state}
    if state["case"]["cache"] == "e4m3":
        return {"q": state["q_out"], "k": state["k_cache"].view(TORCH["e4m3"]), "v": state["v_cache"].view(TORCH["e4m3"]), "k_scale": state["k_scale"], "v_scale": state["v_scale"]}
    return {"q": state["q_out"], "k": state["k_cache"], "v": state["v_cache"]}


# ---- in 64 bits -----------------------------------------------------------------------------------------------------------


def _turned(x, pos, case, inv_freq):
    """One sequence's rows in 64 bits, as complex numbers that are turned by the angle of their position: tokens x heads x head_dim"""
    rot = case["rot"]
    if not rot:
        return x
    flat = x[..., :rot]
    z = torch.complex(flat[..., : rot // 2], flat[..., rot // 2:]) if case["pairs"] == "halves" else torch.view_as_complex(flat.unflatten(-1, (-1, 2)).contiguous())
    angle = pos.double()[:, None, None] * inv_freq.double()
    z = z * torch.polar(torch.ones_like(angle), angle)
    out = x.clone()
    out[..., :rot] = torch.cat([z.real, z.imag], -1) if case["pairs"] == "halves" else torch.view_as_real(z).flatten(-2)
    return out


def _pow2(x):
    """The smallest power of two, at least LOWEST_SCALE, that x is at most 448 times"""
    k = torch.ceil(torch.log2(x.clamp_min(1e-300) / 448))
    k = torch.where(x > 448 * torch.exp2(k), k + 1, torch.where(x <= 448 * torch.exp2(k - 1), k - 1, k))
    return torch.exp2(k).clamp_min(LOWEST_SCALE)


def _exact_append(st):
    c, size = st["case"], st["case"]["page"]
    lens, news = _lengths(c)
    caches = {n: st[n + "_cache"].view(TORCH[c["cache"]]).double() for n in ("k", "v")}
    scales = {n: st[n + "_scale"].double() for n in ("k", "v")} if c["cache"] == "e4m3" else None
    q_out, row = [], 0
    for b, (length, n) in enumerate(zip(lens, news)):
        pos = torch.arange(length - n, length, device="cuda")
        x = st["qkv"][row: row + n].double().view(n, -1, c["head_dim"])
        row += n
        q_out.append(_turned(x[:, : c["heads"]], pos, c, st["inv_freq"]).reshape(n, -1))
        new = {"k": _turned(x[:, c["heads"]: c["heads"] + c["kv_heads"]], pos, c, st["inv_freq"]), "v": x[:, c["heads"] + c["kv_heads"]:]}
        for at in range((length - n) // size, -(-length // size)):
            page = int(st["table"][b, at])
            lo, hi = max(0, length - n - at * size), min(size, length - at * size)
            first = at * size + lo - (length - n)
            for name, x in new.items():
                part = x[first: first + hi - lo].transpose(0, 1)  # kv_heads x tokens x head_dim
                if scales is not None:
                    most, old = part.abs().amax((1, 2)), scales[name][page]
                    scale = _pow2(most) if lo == 0 else torch.where(most > 448 * old, _pow2(most), old)
                    caches[name][page] *= (old / scale)[:, None, None] if lo else 1.0
                    scales[name][page] = scale
                    part = part / scale[:, None, None]
                caches[name][page, :, lo:hi] = part
    got = {"q": torch.cat(q_out), **caches}
    return {**got, "k_scale": scales["k"], "v_scale": scales["v"]} if scales is not None else got


def _exact_attend(st):
    c = st["case"]
    lens, news = _lengths(c)
    group, rows, row = c["heads"] // c["kv_heads"], [], 0
    for b, (length, n) in enumerate(zip(lens, news)):
        table = st["table"][b].long()
        dense = []
        for name in ("k", "v"):
            x = st[name + "_cache"][table].view(TORCH[c["cache"]]).double()
            if c["cache"] == "e4m3":
                x = x * st[name + "_scale"][table].double()[:, :, None, None]
            dense.append(x.transpose(0, 1).flatten(1, 2)[:, :length])
        q = st["q"][row: row + n].double().view(n, c["heads"], c["head_dim"])
        row += n
        heads = []
        for h in range(c["heads"]):
            s = q[:, h] @ dense[0][h // group].t().contiguous() / math.sqrt(c["head_dim"])
            if c["causal"] and n > 1:
                s += torch.full((n, length), -math.inf, dtype=torch.float64, device="cuda").triu(length - n + 1)
            heads.append(torch.softmax(s, -1) @ dense[1][h // group].contiguous())
        rows.append(torch.stack(heads, 1).reshape(n, -1))
    return torch.cat(rows)


def _exact_logprobs(st):
    x = torch.log_softmax(st["logits"].double(), -1)
    tokens = st["tokens"]
    got = {"logprob": torch.where(tokens < 0, 0.0, x[torch.arange(len(tokens), device="cuda"), tokens.clamp_min(0)]), "entropy": torch.special.entr(x.exp()).sum(-1)}
    if st["case"]["top"]:
        values, ids = torch.sort(st["logits"].double(), dim=-1, descending=True, stable=True)
        got["top_ids"] = ids[:, : st["case"]["top"]].to(torch.int32)
        got["top_logprobs"] = x.gather(1, ids[:, : st["case"]["top"]])
    return got


EXACT = {"append": _exact_append, "attend": _exact_attend, "logprobs": _exact_logprobs}


def exact(case, seed):
    return EXACT[case["kind"]](prepare(case, seed))


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------


def work(case):
    if case["kind"] == "logprobs":
        n = float(case["rows"] * case["vocab"])
        return {"bytes": SIZE[case["dtype"]] * n + case["rows"] * (16 + 8 * case["top"]), "flops": 6 * n}
    lens, news = _lengths(case)
    dim, heads, kv_heads, es, cs = case["head_dim"], case["heads"], case["kv_heads"], SIZE[case["dtype"]], SIZE[case["cache"]]
    if case["kind"] == "append":  # rows in; rotated queries out, keys and values into the cache
        t = float(sum(news))
        return {"bytes": t * dim * (heads * 2 * es + kv_heads * 2 * (es + cs)), "flops": t * dim * 3 * (heads + kv_heads)}
    # queries and outputs, and the keys and values that some query sees
    pairs = sum(n * k - (n * (n - 1) / 2 if case["causal"] else 0) for k, n in zip(lens, news))
    return {"bytes": 2.0 * es * sum(news) * heads * dim + 2.0 * cs * sum(lens) * kv_heads * dim, "flops": 4.0 * pairs * heads * dim}
