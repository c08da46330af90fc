"""Operators of a server that answers many requests on one prompt, each as it is measured: its inputs, the call that a
program makes, the same in elementary torch operations, its result in 64 bits, and the work it cannot do without.

Three kinds of case, in the order in which a step meets them:

  tables    `requests` requests bring new tokens: their pages are taken from the pool's free stack, and the step's
            arrays are made (first token, request, position and cache slot of every token, the block tables).
  prefix    attention of the step's tokens over the paged cache, where the requests of a group share the pages of a
            long prefix and each has keys of its own behind it.
  logprobs  log-probability and place of a given token in each row of logits, the row's entropy, and the `top` best
            alternatives.

Sizes: GPT-2 small's and XL's heads and vocabulary, groups of heads on fewer key heads, and generic ones.
"""
import math

import torch

own = False


def listed():
    return [
        # decode of one server: 64 requests bring a token each
        dict(kind="tables", name="tables_decode", requests=64, most=1, context=900, page=16),
        # a step of prompt portions, of every length down to none
        dict(kind="tables", name="tables_prompts", requests=37, most=900, context=700, page=16),
        # a long-document batch: a quarter of a million positions in one step
        dict(kind="tables", name="tables_large", requests=515, most=1024, context=3000, page=64),
        # a few samples of one short prompt at GPT-2 small's heads: latency is all there is
        dict(kind="prefix", name="prefix_small", groups=1, requests=8, tokens=1, prefix=512, own=64, heads=12, kv_heads=12,
             dim=64, page=16, dtype="bfloat16", padded=0),
        # 64 answers drawn from one long document, GPT-2 XL's heads
        dict(kind="prefix", name="prefix_samples", groups=1, requests=64, tokens=1, prefix=8192, own=300, heads=25, kv_heads=25,
             dim=64, page=16, dtype="bfloat16", padded=0),
        # several candidate answers to each of three questions, all their tokens at once
        dict(kind="prefix", name="prefix_scoring", groups=3, requests=23, tokens=37, prefix=1501, own=0, heads=16, kv_heads=16,
             dim=64, page=16, dtype="bfloat16", padded=5),
        # a server's system prompt before 256 conversations, heads in groups of four
        dict(kind="prefix", name="prefix_server", groups=1, requests=256, tokens=1, prefix=32768, own=200, heads=32, kv_heads=8,
             dim=128, page=64, dtype="bfloat16", padded=0),
        # the 32-bit path: two prompts, eleven samples each
        dict(kind="prefix", name="prefix_float32", groups=2, requests=11, tokens=1, prefix=1000, own=100, heads=12, kv_heads=12,
             dim=64, page=16, dtype="float32", padded=0),
        # the token just chosen, with five alternatives, for one request
        dict(kind="logprobs", name="logprobs_one", rows=1, vocab=50257, top=5, allowed=1.0, padding=0, dtype="float32"),
        # a decode step of 64 requests under a grammar that forbids half of the vocabulary
        dict(kind="logprobs", name="logprobs_step", rows=64, vocab=50257, top=20, allowed=0.5, padding=0, dtype="float32"),
        # scoring a prompt: every position of a full step
        dict(kind="logprobs", name="logprobs_prompt", rows=2048, vocab=50257, top=1, allowed=1.0, padding=0, dtype="float32"),
        # bfloat16 logits of a wide vocabulary whose rows are padded
        dict(kind="logprobs", name="logprobs_bfloat16", rows=777, vocab=128000, top=20, allowed=1.0, padding=256, dtype="bfloat16"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["tables", "prefix", "prefix", "prefix", "logprobs", "logprobs"])
    if kind == "tables":
        n = _log(rng, 1, 4096)
        most = 1 if rng.random() < 0.4 else _log(rng, 2, max(2, min(4096, 500000 // n)))
        return dict(kind=kind, requests=n, most=most, context=_log(rng, 1, 4000), page=rng.choice([8, 16, 32, 64, 128]))
    if kind == "logprobs":
        vocab = _log(rng, 200, 200000)
        return dict(kind=kind, rows=_log(rng, 1, min(2048, 100000000 // vocab)), vocab=vocab,
                    top=rng.choice([0, 1, 3, 5, 10, 20, 32]), allowed=rng.choice([1.0, 1.0, 0.5, 0.01]),
                    padding=rng.choice([0, 0, 7, 64]), dtype=rng.choice(["float32", "float32", "bfloat16"]))
    dtype = "float32" if rng.random() < 0.2 else "bfloat16"
    kv_heads = rng.choice([1, 2, 4, 8, 12])
    heads = kv_heads * rng.choice([1, 1, 2, 4, 5, 8])
    groups = rng.choice([1, 1, 2, 5])
    tokens = rng.choice([1, 1, 1, _log(rng, 2, 40)])
    requests = _log(rng, 1, 256 if tokens == 1 else 2000) // (groups * tokens) + 1
    rows = groups * requests * tokens * heads
    cost = 3e7 if dtype == "float32" else 2.5e8                # tokens x heads x prefix
    return dict(kind=kind, groups=groups, requests=requests, tokens=tokens, prefix=_log(rng, 1, max(2, min(32768, cost / rows))),
                own=_log(rng, 1, 400), heads=heads, kv_heads=kv_heads, dim=rng.choice([64, 64, 64, 128, 128, 96]),
                page=rng.choice([16, 16, 16, 32, 64]), dtype=dtype, padded=rng.choice([0, 0, 3]))


# ---------------------------------------------------------------------------------------------------------------- inputs
def _rand(gen):
    def ints(low, high, *shape):
        return torch.randint(low, high, shape, generator=gen, device="cuda", dtype=torch.int32)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")
    return ints, normal


def _lengths(low, high, n):
    """n lengths of low..high that follow from the case alone, so that every seed's outputs have the same sizes."""
    gen = torch.Generator().manual_seed(n * 7919 + high)
    return torch.randint(low, high + 1, (n,), generator=gen, dtype=torch.int32).cuda()


def _cuda_i32(n):
    return torch.zeros(n, dtype=torch.int32, device="cuda")


def _prepare_tables(c, ints):
    R, page = c["requests"], c["page"]
    q_len = _lengths(0 if c["most"] > 1 else 1, c["most"], R)
    kv_len = ints(0, c["context"] + 1, R)
    held = (kv_len + page - 1) // page
    wanted = (kv_len + q_len + page - 1) // page
    T, n_held, n_wanted = (int(x) for x in (q_len.sum(), held.sum(), wanted.sum()))
    width = (c["context"] + c["most"] + page - 1) // page
    n_pages = n_wanted + 100
    order = torch.argsort(ints(0, 1 << 30, n_pages)).to(torch.int32)
    table = torch.full((R, width), -1, dtype=torch.int32, device="cuda")
    table[torch.arange(width, device="cuda")[None, :] < held[:, None]] = order[:n_held]
    return dict(c=c, T=T, q_len=q_len, kv_len=kv_len, free=order[n_held:].clone(), table=table,
                n_free=torch.tensor([n_pages - n_held], dtype=torch.int32, device="cuda"),
                q_start=_cuda_i32(R + 1), new_len=_cuda_i32(R), token_req=_cuda_i32(T), positions=_cuda_i32(T),
                slots=_cuda_i32(T), left=_cuda_i32(1), status=_cuda_i32(1))


def _prepare_prefix(c, ints, normal):
    G, N, page, H, Hkv, D = c["groups"], c["requests"], c["page"], c["heads"], c["kv_heads"], c["dim"]
    dt = getattr(torch, c["dtype"])
    R = G * N
    group_of = torch.arange(R, device="cuda") // N
    # the first group's prefix is the longest; candidate answers have lengths of their own
    shared = ints((c["prefix"] + 1) // 2, c["prefix"] + 1, G)
    shared[0] = c["prefix"]
    n_tok = _lengths((c["tokens"] + 1) // 2, c["tokens"], R)
    before = shared[group_of] + ints(0, c["own"] + 1, R)
    length = before + n_tok
    # whole pages of a prefix are the same in the rows of its group; what it leaves of a page, each row holds for itself
    n_shared = shared // page
    wide = int((length + page - 1).max()) // page
    column = torch.arange(wide, device="cuda")[None, :]
    mine = (column >= n_shared[group_of][:, None]) & (column * page < length[:, None])
    common = column < n_shared[:, None]
    n_common, n_mine = int(common.sum()), int(mine.sum())
    n_pages = n_common + n_mine + 3
    order = torch.argsort(ints(0, 1 << 30, n_pages)).to(torch.int32)
    rows = torch.zeros((G, wide), dtype=torch.int32, device="cuda")
    rows[common] = order[:n_common]
    table = rows[group_of].clone()
    table[mine] = order[n_common:n_common + n_mine]
    cache = normal(n_pages, 2, Hkv, page, D).to(dt)
    cut = torch.nonzero((shared % page != 0)[group_of])[:, 0]
    if cut.numel():
        at = n_shared[group_of[cut]].long()
        kept = (torch.arange(page, device="cuda")[None, :] < (shared % page)[group_of[cut]][:, None])[:, None, None, :, None]
        theirs, first = table[cut, at].long(), table[group_of[cut] * N, at].long()
        cache[theirs] = torch.where(kept, cache[first], cache[theirs])
    T = int(n_tok.sum())
    token_req = torch.repeat_interleave(torch.arange(R, device="cuda"), n_tok.long(), output_size=T)
    ends = torch.cumsum(n_tok, 0)
    place = torch.arange(T, device="cuda") - (ends - n_tok)[token_req]
    group_start = torch.cat([ends.new_zeros(1), ends[N - 1::N]])
    rows_q = T + c["padded"]
    pad = torch.zeros(c["padded"], dtype=torch.int32, device="cuda")
    return dict(c=c, T=T, q=(1.5 * normal(rows_q, H * D)).to(dt), cache=cache, table=table,
                token_req=torch.cat([token_req.to(torch.int32), pad]),
                positions=torch.cat([(before[token_req] + place).to(torch.int32), pad]),
                group_start=group_start.to(torch.int32), shared=shared, scale=1.0 / math.sqrt(D),
                out=torch.zeros((rows_q, H * D), dtype=dt, device="cuda"), longest=c["prefix"],
                most=int(torch.diff(group_start).max()), behind=int((length - shared[group_of]).max()))


def _prepare_logprobs(c, ints, normal):
    n, V, k = c["rows"], c["vocab"], c["top"]
    dt = getattr(torch, c["dtype"])
    x = normal(n, V + c["padding"])
    x = (3.0 * x + 0.5 * x * x).to(dt)                       # a few words stand out, as in a model's logits
    if c["allowed"] < 1.0:
        x[:, ints(0, 1 << 20, V + c["padding"]) >= c["allowed"] * (1 << 20)] = float("-inf")
    if c["padding"]:
        x[:, V:] = float("nan")
    x = x[:, :V]
    tokens = ints(0, V, n)
    likely = torch.arange(n, device="cuda") % 4 != 3          # most given tokens are likely ones, some rows ask for none
    tokens = torch.where(likely, x.float().argmax(1).to(torch.int32), tokens)
    tokens[5::17] = -1
    f32 = dict(dtype=torch.float32, device="cuda")
    return dict(c=c, logits=x, tokens=tokens, logprob=torch.zeros(n, **f32), entropy=torch.zeros(n, **f32), place=_cuda_i32(n),
                top_ids=torch.zeros((n, k), dtype=torch.int32, device="cuda"), top_logprobs=torch.zeros((n, k), **f32))


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    ints, normal = _rand(gen)
    if case["kind"] == "tables":
        return _prepare_tables(case, ints)
    if case["kind"] == "prefix":
        return _prepare_prefix(case, ints, normal)
    return _prepare_logprobs(case, ints, normal)


# ----------------------------------------------------------------------------------------------------------- plain forms
def _plain_tables(s):
    q_len, kv_len, page, T = s["q_len"].long(), s["kv_len"].long(), s["c"]["page"], s["T"]
    end = torch.cumsum(q_len, 0)
    token_req = torch.repeat_interleave(torch.arange(len(q_len), device=end.device), q_len, output_size=T)
    positions = kv_len[token_req] + torch.arange(T, device=end.device) - (end - q_len)[token_req]
    held, wanted = (kv_len + page - 1) // page, (kv_len + q_len + page - 1) // page
    taken = torch.cumsum(wanted - held, 0)
    column = torch.arange(s["table"].shape[1], device=end.device)[None, :]
    nth = (taken - (wanted - held))[:, None] + column - held[:, None]      # which of the step's pages a table entry gets
    fresh = (column >= held[:, None]) & (column < wanted[:, None])
    pages = s["free"][(s["n_free"].long() - 1 - nth).clamp(0, len(s["free"]) - 1)]
    table = torch.where(fresh, pages, s["table"])
    slots = table[token_req, positions // page].long() * page + positions % page
    i32 = torch.int32
    return dict(table=table, q_start=torch.cat([end.new_zeros(1), end]).to(i32), new_len=(kv_len + q_len).to(i32),
                token_req=token_req.to(i32), positions=positions.to(i32), slots=slots.to(i32),
                left=(s["n_free"] - taken[-1]).to(i32), status=torch.zeros_like(s["status"]))


def _softmax_parts(scores, seen):
    """Maximum, exponentials and their sum along the last axis, over the seen entries."""
    scores = torch.where(seen, scores, float("-inf"))
    m = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(torch.isinf(m), 0.0, m))
    return m, e, e.sum(-1, keepdim=True)


def _plain_prefix(s):
    c, T, table = s["c"], s["T"], s["table"].long()
    page, H, Hkv, D = c["page"], c["heads"], c["kv_heads"], c["dim"]
    dev = table.device
    q = s["q"][:T].float().reshape(T, Hkv, H // Hkv, D)
    req, pos, start, shared = s["token_req"][:T].long(), s["positions"][:T].long(), s["group_start"].long(), s["shared"].long()
    # the prefix: every group's tokens against its keys, read through the row of the group's first token
    idx = (start[:-1, None] + torch.arange(s["most"], device=dev)[None, :]).clamp(max=T - 1)
    key = torch.arange(s["longest"], device=dev)
    pages = table[req[start[:-1]]][:, (key // page).clamp(max=table.shape[1] - 1)]
    k, v = (s["cache"][pages, i, :, key % page].float().transpose(1, 2) for i in (0, 1))      # [G, Hkv, L, D]
    qg = q[idx].permute(0, 2, 1, 3, 4)                                                        # [G, Hkv, N, heads a key head, D]
    scores = torch.matmul(qg.reshape(len(shared), Hkv, -1, D), k.transpose(2, 3)).view(*qg.shape[:4], -1) * s["scale"]
    seen = key < torch.minimum(shared[:, None], pos[idx] + 1)[:, :, None]                     # [G, N, L]
    m1, e, l1 = _softmax_parts(scores, seen[:, None, :, None, :])
    o1 = torch.matmul(e.reshape(len(shared), Hkv, -1, e.shape[-1]), v).view_as(qg)
    group = torch.searchsorted(start[1:].contiguous(), torch.arange(T, device=dev), right=True)
    nth = torch.arange(T, device=dev) - start[group]
    m1, l1, o1 = (x.permute(0, 2, 1, 3, 4)[group, nth] for x in (m1, l1, o1))                 # [T, Hkv, heads a key head, ...]
    # the keys behind it, a token's own
    key = shared[group][:, None] + torch.arange(s["behind"], device=dev)[None, :]             # [T, keys]
    pages = torch.gather(table[req], 1, (key // page).clamp(max=table.shape[1] - 1))
    k, v = (s["cache"][pages, i, :, key % page].float().transpose(1, 2) for i in (0, 1))      # [T, Hkv, keys, D]
    m2, e, l2 = _softmax_parts(torch.matmul(q, k.transpose(2, 3)) * s["scale"], (key <= pos[:, None])[:, None, None, :])
    o2 = torch.matmul(e, v)
    m = torch.maximum(m1, m2)
    m = torch.where(torch.isinf(m), 0.0, m)
    f1, f2 = torch.exp(m1 - m), torch.exp(m2 - m)
    total = l1 * f1 + l2 * f2
    out = torch.where(total > 0, (o1 * f1 + o2 * f2) / total, 0.0).reshape(T, H * D)
    s["out"][:T] = out.to(s["out"].dtype)
    return s["out"]


def _plain_logprobs(s):
    x = s["logits"].float()
    V, k = x.shape[1], s["c"]["top"]
    m = x.amax(1, keepdim=True)
    m = torch.where(m == float("-inf"), 0.0, m)               # a row that forbids every word
    e = torch.exp(x - m)
    total = e.sum(1, keepdim=True)
    logp = torch.where(total == 0, float("-inf"), x - m - torch.log(total))
    entropy = -torch.where(e > 0, e * logp, 0.0).sum(1) / torch.where(total == 0, 1.0, total)[:, 0]
    asked = s["tokens"] >= 0
    at = s["tokens"].long().clamp(min=0)[:, None]
    value, index = x.gather(1, at), torch.arange(V, device=x.device)[None, :]
    place = ((x > value) | ((x == value) & (index < at))).sum(1)
    ids = torch.argsort(x, dim=1, descending=True, stable=True)[:, :k]
    return dict(logprob=torch.where(asked, logp.gather(1, at)[:, 0], 0.0), entropy=entropy,
                place=torch.where(asked, place, -1).to(torch.int32), top_ids=ids.to(torch.int32), top_logprobs=logp.gather(1, ids))


def run(state):
    kind = state["c"]["kind"]
    if own:
        return _own(state, kind)
    if kind == "tables":
        return _plain_tables(state)
    if kind == "prefix":
        return _plain_prefix(state)
    return _plain_logprobs(state)


def _own(s, kind):
    from sglang_c_b200.csrc import ops
    if kind == "tables":
        ops.step_tables(s["q_len"], s["kv_len"], s["free"], s["n_free"], s["table"], s["c"]["page"], s["q_start"], s["new_len"],
                        s["token_req"], s["positions"], s["slots"], s["left"], s["status"])
        return {k: s[k] for k in ("table", "q_start", "new_len", "token_req", "positions", "slots", "left", "status")}
    if kind == "prefix":
        ops.attention_prefix(s["q"], s["cache"], s["table"], s["token_req"], s["positions"], s["group_start"], s["shared"],
                             s["out"], s["c"]["heads"], s["scale"], max_own=s["behind"])
        return s["out"]
    ops.token_logprobs(s["logits"], s["tokens"], s["logprob"], entropy=s["entropy"], place=s["place"], top_ids=s["top_ids"],
                       top_logprobs=s["top_logprobs"])
    return {k: s[k] for k in ("logprob", "entropy", "place", "top_ids", "top_logprobs")}


# ------------------------------------------------------------------------------------------------------ results in 64 bits
def _exact_prefix(s):
    c, table, start = s["c"], s["table"].tolist(), s["group_start"].tolist()
    page, H, Hkv, D = c["page"], c["heads"], c["kv_heads"], c["dim"]
    req, pos, shared = s["token_req"].tolist(), s["positions"].tolist(), s["shared"].tolist()
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")

    def rows(r, first, last):
        """Keys and values of request r's positions first .. last-1, [2, kv heads, positions, D]."""
        at = range(first, last)
        pages = torch.tensor([table[r][p // page] for p in at], dtype=torch.long, device="cuda")
        inside = torch.tensor([p % page for p in at], dtype=torch.long, device="cuda")
        return s["cache"][pages, :, :, inside].double().permute(1, 2, 0, 3)

    for g in range(len(shared)):
        if start[g] == start[g + 1]:
            continue
        common = rows(req[start[g]], 0, shared[g])
        mine = {}
        for t in range(start[g], start[g + 1]):
            r = req[t]
            if r not in mine:
                last = max(pos[u] for u in range(start[g], start[g + 1]) if req[u] == r)
                mine[r] = rows(r, shared[g], last + 1)
            n_own = pos[t] + 1 - shared[g]
            q = s["q"][t].double().view(Hkv, H // Hkv, D) * s["scale"]
            k, v = (torch.cat([common[i], mine[r][i, :, :n_own]], 1) for i in (0, 1))
            out[t] = (torch.softmax(q @ k.transpose(1, 2), -1) @ v).reshape(H * D)
    return out


def _exact_logprobs(s):
    rows = []
    for x, t in zip(s["logits"].split(64), s["tokens"].split(64)):
        x = x.double()
        none = (x == float("-inf")).all(1)
        logp = torch.where(none[:, None], x, x - torch.logsumexp(x, 1, keepdim=True))
        entropy = torch.where(none, 0.0, torch.special.entr(torch.softmax(x, 1)).sum(1))
        best = torch.sort(logp, 1, descending=True)[0][:, :s["c"]["top"]]
        rows.append((torch.where(t < 0, 0.0, logp[torch.arange(len(t)), t.long().clamp(min=0)]), entropy, best))
    logprob, entropy, best = (torch.cat(r) for r in zip(*rows))
    return dict(logprob=logprob, entropy=entropy, place=None, top_ids=None, top_logprobs=best)


def exact(case, seed):
    if case["kind"] == "tables":
        return None                                           # whole numbers: the plain form's are exact
    if case["kind"] == "prefix":
        tokens = case["groups"] * case["requests"] * case["tokens"]
        if tokens * case["heads"] * (case["prefix"] + 300) > 4e8 or tokens > 3000:
            return None
        return _exact_prefix(prepare(case, seed))
    return _exact_logprobs(prepare(case, seed))


# ------------------------------------------------------------------------------------------------------------------- work
def work(case):
    c = case
    if c["kind"] == "tables":
        tokens = c["requests"] * (1 if c["most"] == 1 else c["most"] / 2)
        fresh = tokens / c["page"]
        return {"bytes": int(4 * (4 * c["requests"] + 3 * tokens + 2 * fresh)), "flops": int(tokens)}
    if c["kind"] == "prefix":
        size = 4 if c["dtype"] == "float32" else 2
        R = c["groups"] * c["requests"]
        per = (c["tokens"] + (c["tokens"] + 1) // 2) / 2       # tokens of a request, on average
        T, prefix = R * per, c["prefix"] * (0.75 if c["groups"] > 1 else 1.0)
        behind = c["own"] / 2 + per
        kv = 2 * c["kv_heads"] * c["dim"] * size
        return {"bytes": int(kv * (c["groups"] * prefix + R * behind) + 2 * T * c["heads"] * c["dim"] * size),
                "flops": int(4 * c["dim"] * c["heads"] * T * (prefix + c["own"] / 2 + per / 2))}
    size = 4 if c["dtype"] == "float32" else 2
    return {"bytes": int(c["rows"] * (c["vocab"] * size + 4 * (4 + 2 * c["top"]))), "flops": int(4 * c["rows"] * c["vocab"])}
