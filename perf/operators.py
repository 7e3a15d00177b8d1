"""Operators of decoder serving as timed cases: a paged cache of keys and values that is appended to, and the attentions that read it.

A case is a dict of plain values whose "op" names the operator:
  append   Context.kv_append: the new tokens' keys (rotated) and values go to their pages, the queries come back rotated
  paged    Context.attention_paged: each sequence's newest tokens against its keys in the cache
  prefix   Context.attention_prefix: the same where all sequences begin with one shared prefix that is stored once

Sequences: `lens` names how many keys each has after its new tokens ("fixed" or "ragged" up to `most`), `new` how many of them are new
(the queries), "ragged_new" whether prompts differ in length.  Heads: `hq` query heads share `hkv` key heads of width `d`.
"""
import math
import random

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _case(op, dtype, seqs, new, most, lens="fixed", ragged_new=False, hq=32, hkv=8, d=128, page=16, **more):
    return dict(op=op, dtype=dtype, seqs=seqs, new=new, most=most, lens=lens, ragged_new=ragged_new, hq=hq, hkv=hkv, d=d, page=page, **more)


def _append(*a, rotary=128, interleaved=False, source="same", **more):
    return _case("append", *a, rotary=rotary, interleaved=interleaved, source=source, **more)


def _prefix(*a, prefix, **more):
    return _case("prefix", *a, prefix=prefix, **more)


def listed():
    return [
        # one token of one conversation: the smallest call of each generation step
        _append("bf16", 1, 1, 1000, name="append_1_token"),
        # a step of a busy server: one token of each of 256 sequences, interleaved pairs, part of the head rotated
        _append("fp16", 256, 1, 900, lens="ragged", page=24, rotary=64, interleaved=True, name="append_256_tokens"),
        # prompts that arrive together, ragged, from fp32 projections into a cache of halves
        _append("bf16", 5, 2000, 2600, lens="ragged", ragged_new=True, page=64, source="fp32", name="append_prompts"),
        # one conversation, one token: latency
        _case("paged", "bf16", 1, 1, 1500, name="decode_1x1500"),
        # a server's batch of conversations of every length
        _case("paged", "bf16", 64, 1, 8000, lens="ragged", name="decode_64_ragged"),
        # two very long documents, a few draft tokens checked at once
        _case("paged", "fp16", 2, 4, 130001, page=64, name="decode_2x130k_4new"),
        # full precision, the heads of BERT-base, in the framework's own type
        _case("paged", "fp32", 16, 1, 1100, lens="ragged", hq=12, hkv=12, d=64, page=32, name="decode_fp32_16"),
        # prompts read in one go, ragged
        _case("paged", "bf16", 2, 5001, 5001, ragged_new=True, page=16, name="prompts_2x5k"),
        # the next piece of a long prompt, behind what the cache holds
        _case("paged", "fp16", 1, 500, 33000, hq=16, hkv=2, page=128, name="chunk_500_at_33k"),
        # eight samples of one question
        _prefix("bf16", 8, 1, 65, lens="ragged", prefix=1901, name="prefix_8_samples"),
        # a server whose requests share one long instruction
        _prefix("bf16", 128, 1, 500, lens="ragged", prefix=16400, page=32, name="prefix_128_at_16k"),
        # short questions, not yet read, about one shared document
        _prefix("fp16", 16, 60, 60, ragged_new=True, prefix=8200, hq=16, hkv=4, d=64, page=16, name="prefix_16_questions"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(c):  # seconds at this card's rates, about
    w = work(c)
    return max(w["bytes"] / 6.5e12, w["flops"] * (20 if c["dtype"] == "fp32" else 1) / 1.6e15)


def draw(rng):
    while True:
        c = _drawn(rng)
        if _cost(c) <= 160e-6:  # the largest listed ones
            return c


def _drawn(rng):
    op = rng.choice(["append", "paged", "paged", "prefix"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp16", "fp32"])
    hkv, group = rng.choice([1, 2, 4, 8, 12]), rng.choice([1, 2, 4, 5, 8])
    heads = dict(hq=hkv * group, hkv=hkv, d=rng.choice([64, 64, 128, 128, 128, 80, 96, 40]), page=rng.choice([16, 16, 32, 64, 128, 7, 24, 1]))
    lens, ragged_new = rng.choice(["fixed", "ragged"]), rng.random() < 0.5
    if op == "append":
        seqs = _log(rng, 1, 256)
        new = 1 if rng.random() < 0.5 else _log(rng, 1, 8000 // seqs + 1)
        return _append(dtype, seqs, new, new + _log(rng, 1, 1000), lens=lens, ragged_new=ragged_new and new > 1,
                       rotary=rng.choice([heads["d"], heads["d"] // 2, 0]), interleaved=rng.random() < 0.5,
                       source=rng.choice(["same", "fp32"]), **heads)
    slow = 8 if dtype == "fp32" else 1  # what full precision costs beside halves
    if rng.random() < 0.6:  # single tokens, or a few
        seqs, new = _log(rng, 1, 128), rng.choice([1, 1, 1, 2, 5])
        most = _log(rng, new + 1, min(100000, max(64, 300000 // (seqs * slow))))
    else:  # prompts and pieces of prompts
        seqs = _log(rng, 1, 12)
        new = _log(rng, 9, 4000 // seqs // slow + 9)
        most = new + (0 if rng.random() < 0.5 else _log(rng, 1, 16000 // slow))
    if op == "paged":
        return _case("paged", dtype, seqs, new, most, lens=lens, ragged_new=ragged_new and new > 1, **heads)
    return _prefix(dtype, seqs, new, min(most, 2000 + new), lens=lens, ragged_new=ragged_new and new > 1, prefix=_log(rng, 30, 16000 // slow), **heads)


def _shape(c):
    """(keys after the call, new tokens) of each sequence: part of the case, the same for every seed of the data."""
    rng = random.Random(c["seqs"] * 1000003 + c["most"] * 101 + c["new"])
    new = [max(1, int(c["new"] * (1 - 0.6 * rng.random()))) if c["ragged_new"] and i else c["new"] for i in range(c["seqs"])]
    lens = [max(n, int(c["most"] * (1 - 0.9 * rng.random()))) if c["lens"] == "ragged" and i else max(c["most"], n) for i, n in enumerate(new)]
    if c["ragged_new"] and c["most"] == c["new"]:  # prompts from their first token on
        lens = new
    return lens, new


def _angles(c):
    return [10000.0 ** (-2 * j / c["rotary"]) for j in range(c["rotary"] // 2)]


def prepare(case, seed):
    c, g = case, torch.Generator(device="cuda").manual_seed(seed)
    dt = _TYPES[c["dtype"]]
    lens, new = _shape(c)
    per = [-(-n // c["page"]) for n in lens]
    shared = -(-c.get("prefix", 0) // c["page"])
    pages = sum(per) + shared + 3  # a few belong to nobody

    def rand(*shape, dtype=dt):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32 if dtype is torch.float32 else dtype)

    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)  # a server's pages lie in no order
    table = torch.zeros((c["seqs"], max(per)), dtype=torch.int32)
    at = shared
    host = order.cpu()
    for b, n in enumerate(per):
        table[b, :n] = host[at:at + n]
        at += n
    s = dict(case=c, lens=lens, new=new, kv_lens=torch.tensor(lens, dtype=torch.int32).cuda(), table=table.cuda(), prefix_table=order[:shared].contiguous(),
             k_cache=rand(pages, c["page"], c["hkv"], c["d"]), v_cache=rand(pages, c["page"], c["hkv"], c["d"]), q_starts=None)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    s["starts"] = starts
    if len(set(new)) > 1:
        s["q_starts"] = torch.tensor(starts, dtype=torch.int32).cuda()
    if c["op"] == "append":
        # one projection gives queries, keys and values side by side: the operator reads its parts in place
        qkv = rand(starts[-1], c["hq"] + 2 * c["hkv"], c["d"], dtype=torch.float32 if c["source"] == "fp32" else dt)
        s["q"], s["k"], s["v"] = qkv[:, :c["hq"]], qkv[:, c["hq"]:c["hq"] + c["hkv"]], qkv[:, c["hq"] + c["hkv"]:]
        s["inv_freq"] = torch.tensor(_angles(c), dtype=torch.float32).cuda() if c["rotary"] else None
    else:
        s["q"] = rand(starts[-1], c["hq"], c["d"]) * 2  # sharper than uniform: some keys matter more than others
    if own:
        from pet_b200.ops import Context
        s["ctx"] = Context(0)
    return s


def _rotate(x, angle, interleaved, rotary):
    """x [T, H, D] in 32 bits, angle [T, rotary / 2] in 64 bits."""
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    r, rest = x[..., :rotary], x[..., rotary:]
    if interleaved:
        a, b = r[..., 0::2], r[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = r[..., :rotary // 2], r[..., rotary // 2:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, rest), -1)


def _plain_append(s):
    c, dt, dev = s["case"], s["k_cache"].dtype, s["q"].device
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    new = torch.tensor(s["new"], device=dev)
    seq = torch.repeat_interleave(torch.arange(c["seqs"], device=dev), new, output_size=s["starts"][-1])
    first = torch.tensor(s["starts"][:-1], device=dev)
    pos = (s["kv_lens"].long() - new)[seq] + torch.arange(s["starts"][-1], device=dev) - first[seq]
    if s["inv_freq"] is not None:
        angle = pos.double()[:, None] * s["inv_freq"].double()
        q, k = _rotate(q, angle, c["interleaved"], c["rotary"]), _rotate(k, angle, c["interleaved"], c["rotary"])
    page, slot = s["table"][seq, pos // c["page"]].long(), pos % c["page"]
    s["k_cache"][page, slot] = k.to(dt)
    s["v_cache"][page, slot] = v.to(dt)
    return q.to(dt), s["k_cache"], s["v_cache"]


def _plain_attention(s):
    c, dev = s["case"], s["q"].device
    group, scale, out = c["hq"] // c["hkv"], 1.0 / math.sqrt(c["d"]), torch.empty_like(s["q"])
    n0 = c.get("prefix", 0)
    if n0:
        head = s["prefix_table"].long()
        k0, v0 = (x[head].flatten(0, 1)[:n0].float().transpose(0, 1) for x in (s["k_cache"], s["v_cache"]))  # [Hkv, n0, D], for all
    for b, (n, m) in enumerate(zip(s["lens"], s["new"])):
        rows = slice(s["starts"][b], s["starts"][b + 1])
        pages = s["table"][b, :-(-n // c["page"])].long()
        k, v = (x[pages].flatten(0, 1)[:n].float().transpose(0, 1) for x in (s["k_cache"], s["v_cache"]))  # [Hkv, n, D]
        if n0:
            k, v = torch.cat((k0, k), 1), torch.cat((v0, v), 1)
        q = s["q"][rows].float().view(m, c["hkv"], group, c["d"]).permute(1, 2, 0, 3).flatten(1, 2)  # [Hkv, group * m, D]
        ahead = torch.arange(n0 + n, device=dev)[None] > (n0 + n - m + torch.arange(m, device=dev))[:, None]  # [m, keys]: not to be seen
        step = max(1, (1 << 29) // (group * m * (n0 + n)))  # key heads at a time: 2 GB of scores
        parts = []
        for h in range(0, c["hkv"], step):
            x = (q[h:h + step] @ k[h:h + step].transpose(1, 2)).mul_(scale)
            if m > 1:
                x.view(x.shape[0], group, m, -1).masked_fill_(ahead, -math.inf)
            x = x.sub_(x.amax(-1, keepdim=True)).exp_()
            parts.append((x @ v[h:h + step]) / x.sum(-1, keepdim=True))
        y = torch.cat(parts) if len(parts) > 1 else parts[0]
        out[rows] = y.view(c["hkv"], group, m, c["d"]).permute(2, 0, 1, 3).reshape(m, c["hq"], c["d"]).to(out.dtype)
    return out


def run(state):
    s = state
    c = s["case"]
    if not own:
        return _plain_append(s) if c["op"] == "append" else _plain_attention(s)
    ctx = s["ctx"]
    if c["op"] == "append":
        q = ctx.kv_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["kv_lens"], q_starts=s["q_starts"], q=s["q"],
                          inv_freq=s["inv_freq"], interleaved=c["interleaved"])
        return q, s["k_cache"], s["v_cache"]
    if c["op"] == "paged":
        return ctx.attention_paged(s["q"], s["k_cache"], s["v_cache"], s["table"], s["kv_lens"], q_starts=s["q_starts"])
    return ctx.attention_prefix(s["q"], s["k_cache"], s["v_cache"], s["prefix_table"], c["prefix"], s["table"], s["kv_lens"], q_starts=s["q_starts"])


def work(case):
    c = case
    lens, new = _shape(c)
    size, tokens = (4 if c["dtype"] == "fp32" else 2), sum(new)
    index = 4 * (2 * c["seqs"] + sum(-(-n // c["page"]) for n in lens))
    if c["op"] == "append":
        values = tokens * (c["hq"] + 2 * c["hkv"]) * c["d"]
        return {"bytes": values * (size + (4 if c["source"] == "fp32" else size)) + 4 * (tokens + 2 * c["seqs"]), "flops": 3 * tokens * (c["hq"] + c["hkv"]) * c["rotary"]}
    n0 = c.get("prefix", 0)
    pairs = sum(m * (n0 + n) - m * (m - 1) // 2 for n, m in zip(lens, new))
    keys = (n0 + sum(lens)) * c["hkv"] * c["d"] * 2
    return {"bytes": size * (keys + 2 * tokens * c["hq"] * c["d"]) + index, "flops": 4 * pairs * c["hq"] * c["d"]}


def exact(case, seed):
    """The operators token by token and head by head from their definition, in 64 bits."""
    s, c = prepare(case, seed), case
    lens, new = s["lens"], s["new"]

    def where(b, positions):  # rows of the cache that hold these positions of a sequence
        return s["table"][b].long()[positions // c["page"]] * c["page"] + positions % c["page"]

    if c["op"] == "append":
        k_all, v_all = (x.double().reshape(-1, c["hkv"], c["d"]) for x in (s["k_cache"], s["v_cache"]))
        q_all = s["q"].double().clone()
        half = c["rotary"] // 2
        first = torch.arange(half, device="cuda") * (2 if c["interleaved"] else 1)
        second = first + (1 if c["interleaved"] else half)
        for b in range(c["seqs"]):
            rows = slice(s["starts"][b], s["starts"][b + 1])
            pos = torch.arange(lens[b] - new[b], lens[b], device="cuda")
            k = s["k"][rows].double().clone()
            if half:
                z = torch.polar(torch.ones(new[b], half, device="cuda", dtype=torch.float64), pos[:, None] * s["inv_freq"].double()[None])
                for x in (k, q_all[rows]):
                    w = torch.complex(x[..., first], x[..., second]) * z[:, None]
                    x[..., first], x[..., second] = w.real, w.imag
            k_all[where(b, pos)] = k
            v_all[where(b, pos)] = s["v"][rows].double()
        return q_all, k_all.view(s["k_cache"].shape), v_all.view(s["v_cache"].shape)
    n0, group = c.get("prefix", 0), c["hq"] // c["hkv"]
    out = torch.empty(s["q"].shape, device="cuda", dtype=torch.float64)
    flat = [x.view(-1, c["hkv"], c["d"]) for x in (s["k_cache"], s["v_cache"])]
    for b in range(c["seqs"]):
        at = where(b, torch.arange(lens[b], device="cuda"))
        if n0:
            p = torch.arange(n0, device="cuda")
            at = torch.cat((s["prefix_table"].long()[p // c["page"]] * c["page"] + p % c["page"], at))
        seen = n0 + lens[b] - new[b] + 1 + torch.arange(new[b], device="cuda")  # keys that each new token sees
        for j in range(c["hkv"]):
            k, v = (x[at, j].double() for x in flat)
            for h in range(j * group, (j + 1) * group):
                x = s["q"][s["starts"][b]:s["starts"][b + 1], h].double() @ k.T / math.sqrt(c["d"])
                if new[b] > 1:
                    x = x.masked_fill(torch.arange(len(at), device="cuda")[None] >= seen[:, None], -math.inf)
                out[s["starts"][b]:s["starts"][b + 1], h] = torch.softmax(x, -1) @ v
    return out
