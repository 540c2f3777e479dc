"""What a server of decoders needs beside the step of perf/operators.py: matrix products with weights in 4 bits, attention of users
who share a long beginning, and attention over whole prompts that no cache holds.

A case is a dict of plain values.  There are three kinds:

  w4      gp_launch_gemm_w4: rows of activations times a matrix of 4-bit numbers with a scale (and a zero) for each group of a row's values.
  prefix  gp_launch_prefix_attention: the queries of the sequences' last tokens over the pages of a cache, of which the first hold what all
          sequences begin with (a system prompt, a document).
  packed  gp_launch_packed_attention: prompts of different lengths one behind the other, each attending to itself (causal), or the
          sequences of an encoder (not causal).

Where `own` is false the operators are computed in elementary torch operations."""
import math
import random

import torch

own = False

TORCH = {"f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
SIZE = {"f16": 2, "bf16": 2, "e4m3": 1}


def listed():
    gqa = {"heads": 32, "kv_heads": 8, "head_dim": 128}  # four query heads to a head of keys and values
    mha = {"heads": 12, "kv_heads": 12, "head_dim": 64}  # the head layout of the framework's BERT-base
    return [
        # the smallest call: one token through the q, k and v projection of BERT-base's width
        {"name": "w4_one_f16", "kind": "w4", "dtype": "f16", "M": 1, "N": 2304, "K": 768, "group": 64, "zeros": False, "bias": True, "residual": False, "act": "none"},
        # one user's next token through the widest product of a layer
        {"name": "w4_step_bf16", "kind": "w4", "dtype": "bf16", "M": 1, "N": 22528, "K": 4096, "group": 128, "zeros": True, "bias": False, "residual": False, "act": "none"},
        # 24 users' next tokens back to the layer's width, added to what the layer began with
        {"name": "w4_users_f16", "kind": "w4", "dtype": "f16", "M": 24, "N": 4096, "K": 11264, "group": 128, "zeros": True, "bias": False, "residual": True, "act": "none"},
        # the logits of a few users over a vocabulary, the finest groups
        {"name": "w4_vocab_bf16", "kind": "w4", "dtype": "bf16", "M": 5, "N": 131001, "K": 4096, "group": 32, "zeros": False, "bias": False, "residual": False, "act": "none"},
        # a prompt: bound by the matrix products
        {"name": "w4_prompt_bf16", "kind": "w4", "dtype": "bf16", "M": 4001, "N": 8192, "K": 8192, "group": 128, "zeros": False, "bias": False, "residual": False, "act": "none"},
        # the smallest call: three users behind a short instruction
        {"name": "prefix_three_f16", "kind": "prefix", "dtype": "f16", "cache": "f16", **mha, "page": 16, "batch": 3, "new": 1, "shared": 208, "len": 251, "causal": True},
        # a step of 64 users behind a long system prompt, cache in 8 bits: the everyday load of a server
        {"name": "prefix_b64_e4m3", "kind": "prefix", "dtype": "bf16", "cache": "e4m3", **gqa, "page": 64, "batch": 64, "new": 1, "shared": 8192, "len": 10240, "causal": True},
        # a few users with questions about one very long document, with guessed tokens
        {"name": "prefix_document_bf16", "kind": "prefix", "dtype": "bf16", "cache": "bf16", **gqa, "page": 32, "batch": 5, "new": 4, "shared": 131072, "len": 131777, "causal": True},
        # many short answers behind one prompt: bound by the matrix products
        {"name": "prefix_b256_f16", "kind": "prefix", "dtype": "f16", "cache": "f16", **gqa, "page": 64, "batch": 256, "new": 1, "shared": 16384, "len": 16700, "causal": True},
        # the smallest call: one short prompt
        {"name": "packed_one_f16", "kind": "packed", "dtype": "f16", **mha, "batch": 1, "len": 211, "causal": True},
        # texts of all lengths through an encoder without padding: BERT-base's heads, lengths up to that of the heaviest scenario
        {"name": "packed_texts_f16", "kind": "packed", "dtype": "f16", **mha, "batch": 37, "len": 384, "causal": False},
        # long prompts of several users
        {"name": "packed_prompts_bf16", "kind": "packed", "dtype": "bf16", **gqa, "batch": 4, "len": 8192, "causal": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["w4", "w4", "w4", "prefix", "prefix", "prefix", "packed", "packed"])
    dtype = rng.choice(["f16", "bf16"])
    if kind == "w4":
        group = rng.choice([32, 64, 128])
        rows = rng.choice([1, _log(rng, 2, 64), _log(rng, 64, 4001)])
        k = group * max(1, round(_log(rng, 256, 11264) / group))
        n = _log(rng, 200, 131001 if rows <= 64 else 8192)
        return {"kind": kind, "dtype": dtype, "M": rows, "N": n, "K": k, "group": group, "zeros": rng.random() < 0.5, "bias": rng.random() < 0.4,
                "residual": rng.random() < 0.3, "act": rng.choice(["none", "none", "relu", "gelu"])}
    kv_heads, head_dim = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 128])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 8])
    case = {"kind": kind, "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "causal": rng.random() < 0.8}
    if kind == "packed":
        longest = _log(rng, 1, 8192)
        return {**case, "batch": _log(rng, 1, max(1, min(64, 32768 // longest))), "len": longest}
    page, new = rng.choice([16, 32, 64, 128]), rng.choice([1, 1, 1, 2, 5, 17])
    shared = page * max(1, _log(rng, 64, 65536) // page)
    batch = _log(rng, 1, max(1, min(256, 4 * 1024 * 1024 // shared, 256 // new)))
    return {**case, "cache": rng.choice([dtype, "e4m3", "e4m3"]), "page": page, "batch": batch, "new": new, "shared": shared, "len": shared + new + _log(rng, 1, max(2, min(4096, 131072 // batch)))}


def _lengths(case):
    """(tokens in the cache, new tokens) of each sequence; the first has the largest numbers of the case"""
    rng = random.Random(case["batch"] * 1000003 + case["len"] * 1009 + 1)
    if case["kind"] == "packed":
        lens = [case["len"]] + [rng.randint(max(1, case["len"] // 8), case["len"]) for _ in range(case["batch"] - 1)]
        return lens, lens
    lens, news = [case["len"]], [case["new"]]
    for _ in range(case["batch"] - 1):
        n = rng.randint(1, case["new"])
        news.append(n)
        lens.append(rng.randint(case["shared"] + n, case["len"]))
    return lens, news


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# ---- what a program has in hand -----------------------------------------------------------------------------------------


def _prepare_w4(case, gen):
    m, n, k, dtype = case["M"], case["N"], case["K"], TORCH[case["dtype"]]
    groups = k // case["group"]
    st = {"case": case, "a": torch.randn((m, k), generator=gen, device="cuda", dtype=dtype),
          # two numbers to a byte, the even one in the lower half
          "w": torch.randint(0, 256, (n, k // 2), generator=gen, device="cuda", dtype=torch.uint8),
          "scales": ((torch.rand((n, groups), generator=gen, device="cuda") + 0.5) / 64).to(dtype), "zeros": None, "bias": None, "residual": None,
          "c": torch.empty((m, n), device="cuda", dtype=dtype)}
    if case["zeros"]:
        st["zeros"] = torch.randint(5, 12, (n, groups), generator=gen, device="cuda", dtype=torch.uint8)
    if case["bias"]:
        st["bias"] = torch.randn((n,), generator=gen, device="cuda", dtype=dtype)
    if case["residual"]:
        st["residual"] = torch.randn((m, n), generator=gen, device="cuda", dtype=dtype)
    return st


def _scale_of(most):
    """The smallest power of two that brings `most` to at most 448, the largest e4m3 value."""
    m, e = torch.frexp(most)
    return torch.ldexp(torch.ones_like(most), e - 9 + (m > 0.875).to(e.dtype))


def _prepare_prefix(case, gen):
    lens, news = _lengths(case)
    page, batch, common = case["page"], case["batch"], case["shared"] // case["page"]
    width = -(-case["len"] // page)
    pages = common + batch * (width - common) + 3
    # pages lie anywhere in the pool; every sequence's first are those that all share
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.cat([order[:common].expand(batch, common), order[common: common + batch * (width - common)].reshape(batch, width - common)], 1).contiguous()
    st = {"case": case, "batch": batch, "tokens": sum(news), "width": width, "pages": pages, "max_new": max(news), "max_len": max(lens), "kv_len": _ints(lens),
          "start": None if case["new"] == 1 else _ints([sum(news[:i]) for i in range(batch + 1)]), "table": table, "shared_table": order[:common].contiguous()}
    for name in ("k", "v"):
        x = torch.randn((pages, case["kv_heads"], page, case["head_dim"]), generator=gen, device="cuda", dtype=TORCH[case["dtype"]])
        # a head's keys and values have a size of their own
        x *= torch.rand((1, case["kv_heads"], 1, 1), generator=gen, device="cuda", dtype=x.dtype) + 0.5
        if case["cache"] == "e4m3":
            scale = _scale_of(x.abs().amax((2, 3)).float())
            st[name + "_scale"] = scale
            x = (x.float() / scale[:, :, None, None]).to(TORCH["e4m3"]).view(torch.uint8)
        st[name + "_cache"] = x
    st["q"] = torch.randn((st["tokens"], case["heads"] * case["head_dim"]), generator=gen, device="cuda", dtype=TORCH[case["dtype"]])
    st["out"] = torch.empty_like(st["q"])
    return st


def _prepare_packed(case, gen):
    lens, _ = _lengths(case)
    tokens, dim, dtype = sum(lens), case["head_dim"], TORCH[case["dtype"]]
    return {"case": case, "tokens": tokens, "start": _ints([sum(lens[:i]) for i in range(len(lens) + 1)]),
            # a row of the projection: q, k and v of one token
            "qkv": torch.randn((tokens, (case["heads"] + 2 * case["kv_heads"]) * dim), generator=gen, device="cuda", dtype=dtype),
            "out": torch.empty((tokens, case["heads"] * dim), device="cuda", dtype=dtype)}


PREPARE = {"w4": _prepare_w4, "prefix": _prepare_prefix, "packed": _prepare_packed}


def prepare(case, seed):
    return PREPARE[case["kind"]](case, torch.Generator(device="cuda").manual_seed(seed))


# ---- the plain form --------------------------------------------------------------------------------------------------


def _plain_w4(st):
    c = st["case"]
    n, groups = st["scales"].shape
    w = torch.stack([st["w"] & 15, st["w"] >> 4], -1).view(n, groups, c["group"]).float()
    w -= 8.0 if st["zeros"] is None else st["zeros"].float()[..., None]
    w *= st["scales"].float()[..., None]
    y = torch.matmul(st["a"].float(), w.view(n, -1).t())
    if st["bias"] is not None:
        y += st["bias"].float()
    if st["residual"] is not None:
        y += st["residual"].float()
    if c["act"] == "relu":
        y = y.clamp_min(0)
    elif c["act"] == "gelu":
        y = 0.5 * y * (1 + torch.erf(y * 2 ** -0.5))
    st["c"].copy_(y)


def _dense(st, name, table):
    """The pages of tables one behind the other, in fp32: rows of the table x kv_heads x keys x head_dim"""
    table = table.long()
    x = st[name + "_cache"]
    if st["case"]["cache"] == "e4m3":
        x = x[table].view(TORCH["e4m3"]).float() * st[name + "_scale"][table][..., None, None]
    else:
        x = x[table].float()
    return x.transpose(1, 2).flatten(2, 3)


def _plain_prefix(st):
    c = st["case"]
    batch, kv_heads, dim, group, n, shared = st["batch"], c["kv_heads"], c["head_dim"], c["heads"] // c["kv_heads"], st["max_new"], c["shared"]
    start = torch.arange(batch + 1, device="cuda") if st["start"] is None else st["start"].long()
    count, step = start.diff(), torch.arange(n, device="cuda")
    row = (start[:-1, None] + step).clamp_max(st["tokens"] - 1)  # batch x n; those behind a sequence's last are not used
    q = st["q"].float().view(-1, kv_heads, group, dim)[row].permute(0, 2, 1, 3, 4).reshape(batch, kv_heads, n * group, dim)
    # what all share is there once, and all rows of a head are multiplied with it together
    k0, v0 = (_dense(st, name, st["shared_table"][None])[0] for name in ("k", "v"))
    every = q.transpose(0, 1).reshape(kv_heads, batch * n * group, dim)
    s0 = torch.matmul(every, k0.transpose(1, 2)).mul_(dim ** -0.5).view(kv_heads, batch, n * group, -1)
    own_table = st["table"][:, shared // c["page"]:]
    k1, v1 = (_dense(st, name, own_table) for name in ("k", "v"))
    seen = st["kv_len"].long()[:, None] - (count[:, None] - 1 - step if c["causal"] else torch.zeros_like(step)) - shared  # own keys that a query sees
    hidden = torch.arange(k1.shape[2], device="cuda") >= seen.repeat_interleave(group, 1)[:, None, :, None]
    s1 = torch.matmul(q, k1.transpose(2, 3)).mul_(dim ** -0.5).masked_fill_(hidden, -math.inf).transpose(0, 1)
    most = torch.maximum(s0.amax(-1, keepdim=True), s1.amax(-1, keepdim=True))
    s0, s1 = torch.exp_(s0.sub_(most)), torch.exp_(s1.sub_(most))
    o = torch.matmul(s0.view(kv_heads, batch * n * group, -1), v0).view(kv_heads, batch, n * group, dim) + torch.matmul(s1.transpose(0, 1), v1).transpose(0, 1)
    o /= s0.sum(-1, keepdim=True) + s1.sum(-1, keepdim=True)
    o = o.view(kv_heads, batch, n, group, dim).permute(1, 2, 0, 3, 4).reshape(batch, n, -1)
    seq = torch.repeat_interleave(torch.arange(batch, device="cuda"), count, output_size=st["tokens"])
    st["out"].copy_(o[seq, torch.arange(st["tokens"], device="cuda") - start[seq]])


def _plain_packed(st):
    c = st["case"]
    heads, kv_heads, dim = c["heads"], c["kv_heads"], c["head_dim"]
    group, row = heads // kv_heads, 0
    for n in _lengths(c)[0]:
        x = st["qkv"][row: row + n].float().view(n, heads + 2 * kv_heads, dim).transpose(0, 1).contiguous()
        q, k, v = x.split([heads, kv_heads, kv_heads])
        s = torch.matmul(q.reshape(kv_heads, group * n, dim), k.transpose(1, 2)).mul_(dim ** -0.5).view(kv_heads, group, n, n)
        if c["causal"]:
            s.masked_fill_(torch.ones((n, n), dtype=torch.bool, device="cuda").triu_(1), -math.inf)
        s = torch.exp_(s.sub_(s.amax(-1, keepdim=True)))
        o = torch.matmul(s.view(kv_heads, group * n, n), v) / s.sum(-1).view(kv_heads, group * n, 1)
        st["out"][row: row + n] = o.view(heads, n, dim).transpose(0, 1).reshape(n, -1)
        row += n


# ---- the framework's operators ------------------------------------------------------------------------------------------


def _at(x):
    return None if x is None else x.data_ptr()


def _w4_params(gp, st):
    c = st["case"]
    groups = c["K"] // c["group"]
    return gp.GemmW4Params(dtype=gp.DTYPE_BY_NAME[c["dtype"]], M=c["M"], N=c["N"], K=c["K"], group=c["group"], A=_at(st["a"]), lda=c["K"], W=_at(st["w"]), ldw=c["K"] // 2,
                           scales=_at(st["scales"]), ld_scales=groups, zeros=_at(st["zeros"]), ld_zeros=groups, C=_at(st["c"]), ldc=c["N"], bias=_at(st["bias"]),
                           residual=_at(st["residual"]), act={"none": gp.ACT_NONE, "relu": gp.ACT_RELU, "gelu": gp.ACT_GELU}[c["act"]])


def _prefix_params(gp, st):
    c = st["case"]
    e8 = c["cache"] == "e4m3"
    cache = gp.KvCache(dtype=gp.E4M3 if e8 else gp.DTYPE_BY_NAME[c["cache"]], kv_heads=c["kv_heads"], head_dim=c["head_dim"], page_size=c["page"], pages=st["pages"],
                       k=_at(st["k_cache"]), v=_at(st["v_cache"]), k_scale=_at(st["k_scale"]) if e8 else None, v_scale=_at(st["v_scale"]) if e8 else None)
    p = gp.PrefixAttentionParams(shared_len=c["shared"], shared_table=_at(st["shared_table"]), attention=gp.PagedAttentionParams(
        dtype=gp.DTYPE_BY_NAME[c["dtype"]], cache=cache, batch=st["batch"], tokens=st["tokens"], max_new=st["max_new"], max_len=st["max_len"], start=_at(st["start"]),
        kv_len=_at(st["kv_len"]), page_table=_at(st["table"]), table_width=st["width"], heads=c["heads"], q=_at(st["q"]), ld_q=st["q"].shape[1], out=_at(st["out"]),
        ld_out=st["out"].shape[1], scale=c["head_dim"] ** -0.5, causal=int(c["causal"])))
    # what a program allocates once and keeps for its calls: zeroed before the first
    n = gp.C.c_size_t()
    gp.check(gp.lib().gp_prefix_attention_work_bytes(gp.C.byref(p), gp.C.byref(n)))
    st["work"] = torch.zeros(max(1, n.value), dtype=torch.uint8, device="cuda")
    p.attention.work, p.attention.work_bytes = st["work"].data_ptr(), n.value
    return p


def _packed_params(gp, st):
    c = st["case"]
    at, size, ld = st["qkv"].data_ptr(), st["qkv"].element_size() * c["head_dim"], st["qkv"].shape[1]
    return gp.PackedAttentionParams(dtype=gp.DTYPE_BY_NAME[c["dtype"]], batch=c["batch"], tokens=st["tokens"], max_len=c["len"], start=_at(st["start"]), heads=c["heads"],
                                    kv_heads=c["kv_heads"], head_dim=c["head_dim"], q=at, ld_q=ld, k=at + size * c["heads"], v=at + size * (c["heads"] + c["kv_heads"]), ld_kv=ld,
                                    out=_at(st["out"]), ld_out=st["out"].shape[1], scale=c["head_dim"] ** -0.5, causal=int(c["causal"]))


ENTRY = {"w4": ("gp_launch_gemm_w4", _w4_params), "prefix": ("gp_launch_prefix_attention", _prefix_params), "packed": ("gp_launch_packed_attention", _packed_params)}
PLAIN = {"w4": _plain_w4, "prefix": _plain_prefix, "packed": _plain_packed}


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
    return state["c" if kind == "w4" else "out"]


# ---- in 64 bits -----------------------------------------------------------------------------------------------------------


def _exact_w4(st):
    c = st["case"]
    k = torch.arange(c["K"], device="cuda")
    out = []
    for n0 in range(0, c["N"], 8192):  # some of the matrix's rows at a time
        part = slice(n0, n0 + 8192)
        q = (st["w"][part][:, k // 2].int() >> (4 * (k % 2))) % 16
        zero = torch.full_like(q, 8) if st["zeros"] is None else st["zeros"][part][:, k // c["group"]].int()
        w = (q - zero).double() * st["scales"][part].double()[:, k // c["group"]]
        out.append(st["a"].double() @ w.t().contiguous())
    y = torch.cat(out, 1)
    for name in ("bias", "residual"):
        if st[name] is not None:
            y = y + st[name].double()
    return {"none": lambda x: x, "relu": torch.relu, "gelu": torch.nn.functional.gelu}[c["act"]](y)


def _attended(q, k, v, hidden):
    """heads x rows x dim over heads x keys x dim, in 64 bits"""
    s = torch.bmm(q, k.transpose(1, 2).contiguous()) / math.sqrt(q.shape[-1])
    if hidden is not None:
        s = s.masked_fill(hidden, -math.inf)
    return torch.bmm(torch.softmax(s, -1), v)


def _exact_prefix(st):
    c = st["case"]
    lens, news = _lengths(c)
    group, row, rows = c["heads"] // c["kv_heads"], 0, []
    for b, (length, n) in enumerate(zip(lens, news)):
        pages = st["table"][b, : -(-length // c["page"])].long()
        dense = []
        for name in ("k", "v"):
            x = st[name + "_cache"][pages].view(TORCH[c["cache"]]).double()
            if c["cache"] == "e4m3":
                x *= st[name + "_scale"][pages].double()[:, :, None, None]
            dense.append(x.transpose(0, 1).flatten(1, 2)[:, :length].contiguous())
        q = st["q"][row: row + n].double().view(n, c["kv_heads"], group, -1).transpose(0, 1).reshape(c["kv_heads"], n * group, -1)
        row += n
        hidden = None
        if c["causal"] and n > 1:
            hidden = torch.arange(length, device="cuda") > torch.arange(length - n, length, device="cuda").repeat_interleave(group)[:, None]
        rows.append(_attended(q, dense[0], dense[1], hidden).view(c["kv_heads"], n, group, -1).transpose(0, 1).reshape(n, -1))
    return torch.cat(rows)


def _exact_packed(st):
    c = st["case"]
    heads, kv_heads, dim, row, out = c["heads"], c["kv_heads"], c["head_dim"], 0, []
    for n in _lengths(c)[0]:
        x = st["qkv"][row: row + n].double().view(n, -1, dim)
        row += n
        hidden = torch.arange(n, device="cuda") > torch.arange(n, device="cuda")[:, None] if c["causal"] else None
        got = [_attended(x[None, :, h].contiguous(), x[None, :, heads + h * kv_heads // heads].contiguous(), x[None, :, heads + kv_heads + h * kv_heads // heads].contiguous(), hidden)
               for h in range(heads)]
        out.append(torch.cat(got).transpose(0, 1).reshape(n, -1))
    return torch.cat(out)


EXACT = {"w4": _exact_w4, "prefix": _exact_prefix, "packed": _exact_packed}


def exact(case, seed):
    return EXACT[case["kind"]](prepare(case, seed))


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------


def work(case):
    if case["kind"] == "w4":
        m, n, k = float(case["M"]), float(case["N"]), float(case["K"])
        side = k / case["group"] * n * (3 if case["zeros"] else 2) + (2 * n if case["bias"] else 0) + (2 * m * n if case["residual"] else 0)
        return {"bytes": n * k / 2 + side + 2 * m * k + 2 * m * n, "flops": 2 * m * n * k}
    lens, news = _lengths(case)
    dim, heads, kv_heads, es = case["head_dim"], case["heads"], case["kv_heads"], SIZE[case["dtype"]]
    pairs = sum(n * k - (n * (n - 1) / 2 if case["causal"] else 0) for k, n in zip(lens, news))  # of queries and the keys that they see
    if case["kind"] == "packed":
        keys, cs = sum(lens), es
    else:  # what all share once, and what each has of its own
        keys, cs = case["shared"] + sum(n - case["shared"] for n in lens), SIZE[case["cache"]]
    return {"bytes": 2.0 * es * sum(news) * heads * dim + 2.0 * cs * keys * kv_heads * dim, "flops": 4.0 * pairs * heads * dim}
