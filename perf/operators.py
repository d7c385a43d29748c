"""The operators of a serving step around the 8-bit paged key/value cache, and their cases.

  plan     block tables and slot maps from request lengths        (kv_plan)
  write    keys and values into the 8-bit cache                   (kv_write)
  attend   attention over the 8-bit paged cache                   (paged_attention)
  score    log probabilities of given tokens, entropy, top ones   (token_logprobs)
  grad     gradient of those log probabilities and entropies      (token_logprobs_backward)

`run` with own = False computes them in elementary torch operations; with own = True it makes the library's calls."""
import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
TORCH = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
F8 = torch.float8_e4m3fn
E_MIN, E_MAX = -32, 64            # a block's scale is 2^e with e in this range


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # The tables of one decoding step of a small server: eight requests, one token each.
        dict(name="plan_decode_8", op="plan", requests=8, context=900, new=1, block=16, lens=1),
        # A large mixed step: most requests decode, every eighth brings a chunk of its prompt; tens of thousands of tokens.
        dict(name="plan_mixed_2000", op="plan", requests=2000, context=6000, new=301, block=16, lens=2),
        # The new token of each of 64 decoding requests: the block it falls into may need a larger scale.
        dict(name="write_decode_64", op="write", dtype="bf16", requests=64, context=1500, new=1, kv_heads=8, dim=128, block=16, lens=3),
        # Prompts written for the first time, ragged, heads read in place from a wider projection's rows.
        dict(name="write_prompt_f16", op="write", dtype="f16", requests=9, context=100, new=2048, kv_heads=8, dim=128, block=64, lens=4),
        # The smallest attention call: two short conversations, small heads, no grouping.
        dict(name="attend_decode_2", op="attend", dtype="bf16", requests=2, context=333, new=1, kv_heads=8, group=1, dim=64, block=16,
             causal=True, lens=5),
        # A server's usual decoding step: 64 ragged requests, four query heads to a key head.
        dict(name="attend_decode_64", op="attend", dtype="bf16", requests=64, context=8000, new=1, kv_heads=8, group=4, dim=128, block=16,
             causal=True, lens=6),
        # One long document: all the work is along one sequence.
        dict(name="attend_long_f16", op="attend", dtype="f16", requests=1, context=131085, new=1, kv_heads=8, group=4, dim=128, block=64,
             causal=True, lens=7),
        # Chunks of prompts behind what the cache holds already: many query rows, bound by the products.
        dict(name="attend_chunk", op="attend", dtype="bf16", requests=4, context=5000, new=2048, kv_heads=8, group=4, dim=128, block=32,
             causal=True, lens=8),
        # The scores that one decoding step returns with its tokens.
        dict(name="score_step_16", op="score", dtype="f32", rows=16, vocab=32768, top=8),
        # Prompt scoring: thousands of positions over a large vocabulary.
        dict(name="score_prompt", op="score", dtype="bf16", rows=2048, vocab=131072, top=20),
        # Policy gradients of a short answer, a vocabulary of odd length.
        dict(name="grad_short_f32", op="grad", dtype="f32", rows=61, vocab=50001),
        # The same for a batch of long answers.
        dict(name="grad_batch", op="grad", dtype="bf16", rows=2048, vocab=131072),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "write", "attend", "attend", "score", "grad"])
    lens = rng.randrange(100, 1 << 20)
    if op == "plan":
        requests = _log(rng, 1, 2000)
        return dict(op=op, requests=requests, context=_log(rng, 1, 6000), new=_log(rng, 1, min(2048, 600000 // requests)),
                    block=rng.choice([16, 32, 64, 128]), lens=lens)
    if op == "write":
        requests, heads, dim = _log(rng, 1, 200), rng.choice([1, 2, 4, 8]), rng.choice([64, 128])
        return dict(op=op, dtype=rng.choice(["bf16", "f16"]), requests=requests, context=_log(rng, 1, 3000),
                    new=1 if rng.random() < 0.4 else _log(rng, 1, max(1, min(2048, 16000 // requests))), kv_heads=heads, dim=dim,
                    block=rng.choice([16, 32, 64, 128]), lens=lens)
    if op == "attend":
        heads, group, dim = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 5, 8]), rng.choice([64, 128])
        kind = rng.choice(["decode", "decode", "several", "chunk"])
        requests = _log(rng, 1, 200 if kind != "chunk" else 8)
        longest = max(64, min(131072, (1 << 22) // (heads * requests)))
        new = 1 if kind == "decode" else rng.randint(2, 8)
        if kind == "chunk":
            new = _log(rng, 9, min(2048, math.isqrt((1 << 29) // (heads * group * requests))))
            longest = max(64, min(longest, (1 << 28) // (heads * group * requests * new)))
        return dict(op=op, dtype=rng.choice(["bf16", "f16"]), requests=requests, context=_log(rng, 16, longest), new=new, kv_heads=heads,
                    group=group, dim=dim, block=rng.choice([16, 32, 64, 128]), causal=rng.random() < 0.8, lens=lens)
    vocab = _log(rng, 1000, 131072)
    rows = _log(rng, 1, min(4000, 200_000_000 // vocab))
    case = dict(op=op, dtype=rng.choice(["bf16", "f16", "f32"]), rows=rows, vocab=vocab)
    return dict(case, top=rng.randint(0, 32)) if op == "score" else case


def _lens(case):
    """(tokens already cached, tokens of this step) of each request."""
    rng = random.Random(case["lens"])
    n, most, new = case["requests"], case["context"], case["new"]
    if n == 1:
        return [most], [new]
    before = [rng.randint(max(0, most // 20), most) for _ in range(n)]
    if case["op"] == "write" and new > 1:                      # prompts: some start, some go on
        before = [0 if rng.random() < 0.6 else b for b in before]
    if case["op"] == "plan" and new > 1:                       # a mixed step
        return before, [rng.randint(max(1, new // 2), new) if i % 8 == 0 else 1 for i in range(n)]
    return before, [rng.randint(max(1, new // 2), new) for _ in range(n)] if new > 8 else [new] * n


def _blocks(tokens, block):
    return -(-tokens // block)


def _tables(case, extra=7):
    """The pool's size, each request's blocks before the step and the list of unused ones (a pool that has been in use: in no order)."""
    before, new = _lens(case)
    bs = case["block"]
    held = [_blocks(b, bs) for b in before]
    total = sum(_blocks(b + n, bs) for b, n in zip(before, new)) + extra
    order = list(range(total))
    random.Random(case["lens"] + 1).shuffle(order)
    rows, at = [], 0
    for h in held:
        rows.append(order[at:at + h])
        at += h
    width = max(_blocks(b + n, bs) for b, n in zip(before, new))
    table = torch.full((case["requests"], width), -1, dtype=torch.int32)
    for r, ids in enumerate(rows):
        table[r, :len(ids)] = torch.tensor(ids, dtype=torch.int32)
    return before, new, total, table, torch.tensor(order[at:], dtype=torch.int32)


def _filled(case):
    """The tables after the step, with the slot of each new token."""
    before, new, total, table, free = _tables(case)
    bs, used = case["block"], 0
    free = free.tolist()
    slots = []
    for r, (b, n) in enumerate(zip(before, new)):
        for j in range(_blocks(b, bs), _blocks(b + n, bs)):
            table[r, j] = free[len(free) - 1 - used]
            used += 1
        pos = torch.arange(b, b + n)
        slots.append(table[r].long()[pos // bs] * bs + pos % bs)
    return before, new, total, table, torch.cat(slots)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _starts(new):
    return _int32([0] + np.cumsum(new).tolist())


def _cache(total, case, g):
    """Codes and scales of a pool in use: values of about unit size, each block and head with a scale of its own."""
    shape = (total, case["kv_heads"], case["block"], case["dim"])
    codes = torch.randn(shape, device=DEV, generator=g, dtype=torch.float16).mul_(96).clamp_(-448, 448).to(F8)
    exps = torch.randint(-8, -5, shape[:2], device=DEV, generator=g)
    return codes, torch.exp2(exps.float())


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    op, st = case["op"], dict(case=dict(case))
    if op == "plan":
        before, new, total, table, free = _tables(case)
        # another seed deals the pool's blocks out differently
        deal = torch.randperm(total, device=DEV, generator=g).int()
        table, free = table.to(DEV), deal[free.to(DEV).long()]
        st.update(context_lens=_int32(before), new_lens=_int32(new), free=free.contiguous(), pool=total, tokens=sum(new),
                  table=torch.where(table >= 0, deal[table.clamp(min=0).long()], table).contiguous(), free_count=_int32([free.numel()]))
        r, t = case["requests"], sum(new)
        st["out"] = dict(query_start=torch.empty(r + 1, dtype=torch.int32, device=DEV), seq_lens=torch.empty(r, dtype=torch.int32, device=DEV),
                         slot_map=torch.empty(t, dtype=torch.int64, device=DEV), positions=torch.empty(t, dtype=torch.int32, device=DEV),
                         token_request=torch.empty(t, dtype=torch.int32, device=DEV), result=torch.empty(4, dtype=torch.int32, device=DEV),
                         free_count=torch.empty(1, dtype=torch.int32, device=DEV))      # apart, so that a step can be planned again
        return st
    if op == "write":
        before, new, total, table, slots = _filled(case)
        heads, dim, t, td = case["kv_heads"], case["dim"], sum(new), TORCH[case["dtype"]]
        rows = torch.randn((t, 3 * heads * dim), device=DEV, generator=g, dtype=torch.float32)       # a projection's rows: queries, keys, values
        rows *= torch.exp2(torch.randint(-3, 4, (t, 1), device=DEV, generator=g).float())            # tokens differ in size
        rows = rows.to(td)
        st.update(k=rows[:, heads * dim:2 * heads * dim], v=rows[:, 2 * heads * dim:], slots=slots.to(DEV), pool=total)
        st["k_cache"], st["k_scale"] = _cache(total, case, g)
        st["v_cache"], st["v_scale"] = _cache(total, case, g)
        return st
    if op == "attend":
        before, new, total, table, _ = _filled(case)
        heads, td = case["kv_heads"] * case["group"], TORCH[case["dtype"]]
        st.update(before=before, new=new, table=table.to(DEV), query_start=_starts(new), pool=total,
                  seq_lens=_int32([b + n for b, n in zip(before, new)]), max_query=max(new), scale=case["dim"] ** -0.5,
                  q=(2 * torch.randn((sum(new), heads, case["dim"]), device=DEV, generator=g)).to(td))
        st["k_cache"], st["k_scale"] = _cache(total, case, g)
        st["v_cache"], st["v_scale"] = _cache(total, case, g)
        st["out"] = torch.empty_like(st["q"])
        st["lse"] = torch.empty((sum(new), heads), dtype=torch.float32, device=DEV)
        return st
    rows, vocab = case["rows"], case["vocab"]
    logits = (3 * torch.randn((rows, vocab), device=DEV, generator=g)).to(TORCH[case["dtype"]])
    logits[:, 7::97] = -math.inf                                                  # tokens that a grammar or a filter has ruled out
    tokens = torch.randint(0, vocab, (rows,), device=DEV, generator=g).int()
    tokens = torch.where(tokens % 97 == 7, tokens - 1, tokens)
    st.update(logits=logits, tokens=tokens)
    if op == "score":
        k = case["top"]
        st["out"] = dict(logprob=torch.empty(rows, device=DEV), entropy=torch.empty(rows, device=DEV), lse=torch.empty(rows, device=DEV),
                         top_ids=torch.empty((rows, k), dtype=torch.int32, device=DEV), top_logprobs=torch.empty((rows, k), device=DEV))
        return st
    # what the forward pass left: the row's log-sum-exp and entropy
    lse, ent = torch.empty(rows, device=DEV), torch.empty(rows, device=DEV)
    for a in range(0, rows, 256):
        x = logits[a:a + 256].double()
        z = torch.logsumexp(x, 1, keepdim=True)
        lse[a:a + 256] = z[:, 0].float()
        ent[a:a + 256] = -((x - z).exp() * torch.where(x == -math.inf, 0.0, x - z)).sum(1).float()
    st.update(lse=lse, entropy=ent, grad_logprob=torch.randn(rows, device=DEV, generator=g), out=torch.empty_like(logits),
              grad_entropy=0.1 * torch.randn(rows, device=DEV, generator=g))
    return st


# ---------------------------------------------------------------------------------------------------------- plain forms
def _plan(st):
    bs, c, n = st["case"]["block"], st["context_lens"].long(), st["new_lens"].long()
    have = (c + bs - 1) // bs
    need = (c + n + bs - 1) // bs - have
    first = torch.cumsum(need, 0) - need
    start = torch.cumsum(n, 0) - n
    column = torch.arange(st["table"].shape[1], device=DEV)[None]
    fresh = (column >= have[:, None]) & (column < (have + need)[:, None])
    taken = (st["free_count"].long() - 1 - first[:, None] - (column - have[:, None])).clamp(0, st["free"].numel() - 1)
    table = torch.where(fresh, st["free"][taken], st["table"])
    t = torch.arange(st["tokens"], device=DEV)
    req = torch.searchsorted((start + n).contiguous(), t, right=True)
    pos = c[req] + t - start[req]
    slots = table[req, pos // bs].long() * bs + pos % bs
    total = need.sum()
    zero = torch.zeros((), dtype=torch.int64, device=DEV)
    return dict(table=table, query_start=torch.cat([start, (start[-1] + n[-1])[None]]).int(), seq_lens=(c + n).int(), slot_map=slots,
                positions=pos.int(), token_request=req.int(), free_count=(st["free_count"] - total).int(),
                result=torch.stack([zero, n.sum(), total, zero]).int())


def _scale_for(amax):
    """The smallest power of two that brings amax to 448 or less."""
    m, e = torch.frexp(amax / 448)
    e = torch.where(m == 0.5, e - 1, e)
    return torch.exp2(torch.where(amax > 0, e, E_MIN).clamp(E_MIN, E_MAX).float())


def _write_one(x, slots, codes, scale, bs):
    total, heads, _, dim = codes.shape
    x = x.reshape(x.shape[0], heads, dim).float()
    blk, off = slots // bs, slots % bs
    amax = torch.zeros((total, heads), device=DEV).index_reduce_(0, blk, x.abs().amax(2), "amax")
    first = torch.full((total,), bs, device=DEV).index_reduce_(0, blk, off, "amin")
    touched = torch.unique(blk)
    old, first = scale[touched], first[touched]
    new = _scale_for(amax[touched])
    new = torch.where((first > 0)[:, None], torch.maximum(old, new), new)
    held = codes[touched].float()
    again = (held * (old / new)[:, :, None, None]).clamp(-448, 448)
    earlier = torch.arange(bs, device=DEV)[None, None, :, None] < first[:, None, None, None]
    codes[touched] = torch.where(earlier, again, held).to(F8)
    scale[touched] = new
    codes.view(torch.uint8)[blk, :, off] = (x / scale[blk][:, :, None]).clamp(-448, 448).to(F8).view(torch.uint8)


def _write(st):
    bs = st["case"]["block"]
    _write_one(st["k"], st["slots"], st["k_cache"], st["k_scale"], bs)
    _write_one(st["v"], st["slots"], st["v_cache"], st["v_scale"], bs)
    return dict(k_cache=st["k_cache"], v_cache=st["v_cache"], k_scale=st["k_scale"], v_scale=st["v_scale"])


def _attend(st):
    c = st["case"]
    bs, heads, group, dim = c["block"], c["kv_heads"], c["group"], c["dim"]
    r, mq = c["requests"], st["max_query"]
    idx = st["table"].clamp(min=0).long()
    n = idx.shape[1] * bs

    def dense(codes, scale):
        x = codes.view(torch.uint8)[idx].view(F8).float() * scale[idx][..., None, None]       # [requests, blocks, heads, block, dim]
        return x.permute(0, 2, 1, 3, 4).reshape(r, heads, n, dim)

    lens, start = st["seq_lens"].long(), st["query_start"].long()
    count = start[1:] - start[:-1]
    key = torch.arange(n, device=DEV)
    k = dense(st["k_cache"], st["k_scale"])
    at = torch.arange(mq, device=DEV)
    rows = (start[:-1, None] + at).clamp(max=st["q"].shape[0] - 1)
    q = st["q"].float()[rows].reshape(r, mq, heads, group, dim).permute(0, 2, 3, 1, 4).reshape(r, heads, group * mq, dim)
    s = (q @ k.transpose(2, 3)).mul_(st["scale"]).reshape(r, heads, group, mq, n)
    del k
    limit = (lens - count)[:, None] + at + 1 if c["causal"] else lens[:, None].expand(r, mq)
    seen = key < torch.minimum(limit, lens[:, None])[:, :, None]                              # [requests, rows, keys]
    s.masked_fill_(~seen[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = s.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    v = torch.where((key < lens[:, None])[:, None, :, None], dense(st["v_cache"], st["v_scale"]), 0.0)
    o = (p.reshape(r, heads, group * mq, n) @ v).reshape(r, heads, group, mq, dim) / torch.where(total > 0, total, 1.0)
    lse = (m + total.log())[..., 0]
    real = at < count[:, None]
    o = o.permute(0, 3, 1, 2, 4).reshape(r, mq, heads * group, dim)[real]
    return dict(out=o.to(st["q"].dtype), lse=lse.permute(0, 3, 1, 2).reshape(r, mq, heads * group)[real])


def _score(st):
    x, k = st["logits"].float(), st["case"]["top"]
    m = x.amax(1, keepdim=True)
    e = (x - m).exp()
    s = e.sum(1, keepdim=True)
    lse = m + s.log()
    y = torch.where(x == -math.inf, 0.0, x - m)
    entropy = (s.log() - (e * y).sum(1, keepdim=True) / s)[:, 0]
    logprob = (x.gather(1, st["tokens"].long()[:, None]) - lse)[:, 0]
    # largest value first, ties by the lower index: one whole number orders both
    bits = (x + 0.0).view(torch.int32).long()
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)
    key = order * (1 << 20) + ((1 << 20) - 1 - torch.arange(x.shape[1], device=DEV))
    ids = ((1 << 20) - 1 - torch.topk(key, k, 1).values % (1 << 20)) if k else st["out"]["top_ids"].long()
    return dict(logprob=logprob, entropy=entropy, lse=lse[:, 0], top_ids=ids.int(), top_logprobs=x.gather(1, ids) - lse)


def _grad(st):
    x = st["logits"].float()
    lp = x - st["lse"][:, None]
    p = lp.exp()
    lp = torch.where(x == -math.inf, 0.0, lp)
    d = -p * (st["grad_logprob"][:, None] + st["grad_entropy"][:, None] * (lp + st["entropy"][:, None]))
    d[torch.arange(x.shape[0], device=DEV), st["tokens"].long()] += st["grad_logprob"]
    return d.to(st["logits"].dtype)


# ---------------------------------------------------------------------------------------------------- the library's calls
def _own(st):
    from pyc_b200 import abi, backend
    kinds = {"bf16": abi.DTYPE_BF16, "f16": abi.DTYPE_F16, "f32": abi.DTYPE_F32}
    c, op = st["case"], st["case"]["op"]
    stream = torch.cuda.current_stream().cuda_stream
    if op == "plan":
        o, table = st["out"], st["table"]
        backend.kv_plan(c["requests"], c["block"], table.shape[1], st["tokens"], st["pool"], st["context_lens"].data_ptr(),
                        st["new_lens"].data_ptr(), st["free"].data_ptr(), st["free_count"].data_ptr(), table.data_ptr(), o["query_start"].data_ptr(),
                        o["seq_lens"].data_ptr(), o["slot_map"].data_ptr(), o["positions"].data_ptr(), o["token_request"].data_ptr(),
                        o["result"].data_ptr(), free_count_out=o["free_count"].data_ptr(), stream=stream)
        return dict(o, table=table)
    if op == "write":
        k, v = st["k"], st["v"]
        backend.kv_write(kinds[c["dtype"]], k.shape[0], c["kv_heads"], c["dim"], c["block"], st["pool"], k.data_ptr(), v.data_ptr(),
                         st["slots"].data_ptr(), st["k_cache"].data_ptr(), st["v_cache"].data_ptr(), st["k_scale"].data_ptr(),
                         st["v_scale"].data_ptr(), k_stride=k.stride(0), v_stride=v.stride(0), stream=stream)
        return dict(k_cache=st["k_cache"], v_cache=st["v_cache"], k_scale=st["k_scale"], v_scale=st["v_scale"])
    if op == "attend":
        heads = c["kv_heads"] * c["group"]
        if "workspace" not in st:       # made once, as a server does
            st["workspace"] = torch.zeros(backend.paged_attention_workspace_bytes(c["requests"], st["max_query"], heads, c["kv_heads"], c["dim"]),
                                          dtype=torch.uint8, device=DEV)
        backend.paged_attention(kinds[c["dtype"]], c["requests"], st["max_query"], heads, c["kv_heads"], c["dim"], c["block"], st["pool"],
                                st["table"].shape[1], st["q"].data_ptr(), st["k_cache"].data_ptr(), st["v_cache"].data_ptr(),
                                st["k_scale"].data_ptr(), st["v_scale"].data_ptr(), st["table"].data_ptr(), st["query_start"].data_ptr(),
                                st["seq_lens"].data_ptr(), st["out"].data_ptr(), st["scale"], c["causal"], st["workspace"].data_ptr(),
                                st["workspace"].numel(), lse=st["lse"].data_ptr(), stream=stream)
        return dict(out=st["out"], lse=st["lse"])
    if op == "score":
        o = st["out"]
        backend.token_logprobs(kinds[c["dtype"]], c["rows"], c["vocab"], st["logits"].data_ptr(), st["tokens"].data_ptr(), o["logprob"].data_ptr(),
                               entropy=o["entropy"].data_ptr(), lse=o["lse"].data_ptr(), top_k=c["top"], top_ids=o["top_ids"].data_ptr(),
                               top_logprobs=o["top_logprobs"].data_ptr(), stream=stream)
        return o
    backend.token_logprobs_backward(kinds[c["dtype"]], c["rows"], c["vocab"], st["logits"].data_ptr(), st["tokens"].data_ptr(), st["lse"].data_ptr(),
                                    st["entropy"].data_ptr(), st["grad_logprob"].data_ptr(), st["grad_entropy"].data_ptr(), st["out"].data_ptr(),
                                    stream=stream)
    return st["out"]


def run(state):
    if own:
        return _own(state)
    return dict(plan=_plan, write=_write, attend=_attend, score=_score, grad=_grad)[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------------------------------ work
def work(case):
    op = case["op"]
    if op == "plan":
        before, new = _lens(case)
        fresh = sum(_blocks(b + n, case["block"]) - _blocks(b, case["block"]) for b, n in zip(before, new))
        return dict(bytes=case["requests"] * 16 + fresh * 8 + sum(new) * 16 + 24, flops=sum(new))
    if op == "write":
        before, new = _lens(case)
        values = sum(new) * case["kv_heads"] * case["dim"] * 2
        touched = sum(_blocks(b + n, case["block"]) - b // case["block"] for b, n in zip(before, new))
        return dict(bytes=values * 3 + sum(new) * 8 + touched * case["kv_heads"] * 16, flops=2 * values)
    if op == "attend":
        before, new = _lens(case)
        heads, dim = case["kv_heads"], case["dim"]
        keys = sum(b + n for b, n in zip(before, new))
        pairs = sum(n * (b + n) - (n * (n - 1) // 2 if case["causal"] else 0) for b, n in zip(before, new))
        rows = sum(new) * heads * case["group"]
        scales = sum(_blocks(b + n, case["block"]) for b, n in zip(before, new)) * (heads * 8 + 4)
        return dict(bytes=2 * keys * heads * dim + rows * (4 * dim + 4) + scales, flops=4 * pairs * heads * case["group"] * dim)
    size = 4 if case["dtype"] == "f32" else 2
    n = case["rows"] * case["vocab"]
    if op == "score":
        return dict(bytes=n * size + case["rows"] * (16 + 8 * case["top"]), flops=5 * n)
    return dict(bytes=2 * n * size + case["rows"] * 20, flops=6 * n)


# ------------------------------------------------------------------------------------------- the definition, in 64 bits
def _codes64():
    """The value of each of the 256 codes: sign, four exponent bits (bias 7), three mantissa bits, no infinities."""
    v = []
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        x = math.nan if (e, m) == (15, 7) else m * 2.0 ** -9 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        v.append(-x if c & 128 else x)
    return torch.tensor(v, dtype=torch.float64, device=DEV)


def _exact_attend(st):
    c, value = st["case"], _codes64()
    bs, heads, group, dim = c["block"], c["kv_heads"], c["group"], c["dim"]
    outs, lses, row = [], [], 0
    for r, (b, n) in enumerate(zip(st["before"], st["new"])):
        length = b + n
        ids = st["table"][r, :_blocks(length, bs)].long()
        q = st["q"][row:row + n].double().reshape(n, heads, group, dim)
        row += n
        o, z = torch.empty((n, heads, group, dim), dtype=torch.float64, device=DEV), torch.empty((n, heads, group), dtype=torch.float64, device=DEV)
        for h in range(heads):
            k, v = ((value[codes[ids, h].view(torch.uint8).long()] * scale[ids, h].double()[:, None, None]).reshape(-1, dim)[:length]
                    for codes, scale in ((st["k_cache"], st["k_scale"]), (st["v_cache"], st["v_scale"])))
            s = torch.einsum("ngd,kd->ngk", q[:, h], k) * st["scale"]
            if c["causal"]:
                late = torch.arange(length, device=DEV) > b + torch.arange(n, device=DEV)[:, None]
                s = s.masked_fill(late[:, None], -math.inf)
            z[:, h] = torch.logsumexp(s, 2)
            o[:, h] = torch.einsum("ngk,kd->ngd", (s - z[:, h][..., None]).exp(), v)
        outs.append(o.reshape(n, heads * group, dim))
        lses.append(z.reshape(n, heads * group))
    return dict(out=torch.cat(outs), lse=torch.cat(lses))


def _exact_write(st):
    value = _codes64()
    whole = value[:127]                                                    # 0 ... 448, ascending
    between = (whole[1:] + whole[:-1]) / 2

    def encode(x):                                                         # to the nearest value, ties to the even code
        a = x.abs().clamp(max=448.0)
        up, down = torch.searchsorted(between, a, right=True), torch.searchsorted(between, a)
        i = torch.where((up != down) & (up % 2 == 1), down, up)
        return torch.copysign(whole[i], x)

    bs, slots = st["case"]["block"], st["slots"].tolist()
    runs = []                                                              # (first token, tokens) that fall into one block
    for t, s in enumerate(slots):
        if t and s == slots[t - 1] + 1 and s % bs:
            runs[-1][1] += 1
        else:
            runs.append([t, 1])
    done = {}
    for name in "kv":
        x, codes, scale = st[name], st[name + "_cache"], st[name + "_scale"].double()
        heads, dim = codes.shape[1], codes.shape[3]
        x = x.double().reshape(-1, heads, dim)
        vals = value[codes.view(torch.uint8).long()]
        for t, n in runs:
            blk, off = slots[t] // bs, slots[t] % bs
            part = x[t:t + n].permute(1, 0, 2)
            need = part.abs().amax((1, 2)) / 448
            e = torch.ceil(torch.log2(need)).clamp(E_MIN, E_MAX)
            e = torch.where(torch.exp2(e - 1) >= need, e - 1, e).clamp(E_MIN, E_MAX)
            s = torch.exp2(torch.where(need > 0, e, float(E_MIN)))
            if off:
                s = torch.maximum(s, scale[blk])
                vals[blk, :, :off] = encode(vals[blk, :, :off] * (scale[blk] / s)[:, None, None])
            vals[blk, :, off:off + n] = encode(part / s[:, None, None])
            scale[blk] = s
        done[name + "_cache"], done[name + "_scale"] = vals, scale
    return done


def exact(case, seed):
    if case["op"] == "plan":
        return None                                                        # whole numbers
    if case["op"] == "attend" and work(case)["flops"] > 3e12:
        return None
    st = prepare(case, seed)
    if case["op"] == "attend":
        return _exact_attend(st)
    if case["op"] == "write":
        return _exact_write(st)
    parts = []
    for a in range(0, case["rows"], 128):
        x, tok = st["logits"][a:a + 128].double(), st["tokens"][a:a + 128].long()
        if case["op"] == "score":
            z = torch.logsumexp(x, 1)
            lp = x - z[:, None]
            h = -torch.xlogy(lp.exp(), lp.exp()).sum(1)
            ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :case["top"]]
            parts.append((lp.gather(1, tok[:, None])[:, 0], h, z, lp.gather(1, ids)))
            continue
        z, h = st["lse"][a:a + 128].double(), st["entropy"][a:a + 128].double()
        u, w = st["grad_logprob"][a:a + 128].double(), st["grad_entropy"][a:a + 128].double()
        p = (x - z[:, None]).exp()
        hot = torch.nn.functional.one_hot(tok, case["vocab"]).double()
        parts.append((hot - p) * u[:, None] - w[:, None] * (torch.xlogy(p, p) + p * h[:, None]))
    if case["op"] == "grad":
        return torch.cat([p.to(torch.float64) for p in parts])
    lp, h, z, top = (torch.cat(x) for x in zip(*parts))
    return dict(logprob=lp, entropy=h, lse=z, top_ids=None, top_logprobs=top)
