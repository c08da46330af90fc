"""Inputs and 64-bit results of the operators for many requests on one prompt (step_tables, attention_prefix, token_logprobs):
plain loops, written from the definitions; no code of the package but its host-side page pool."""
import math

import torch

from sglang_c_b200.cache.pages import PagePool


def tables_by_hand(q_len, kv_len, page, seed=0, spare=5):
    """What step_tables is given and has to give, from the host's page pool, taken request by request."""
    need = [(k + q + page - 1) // page for q, k in zip(q_len, kv_len)]
    held = [(k + page - 1) // page for k in kv_len]
    pool = PagePool(sum(need) + spare)
    order = torch.randperm(pool.n_pages, generator=torch.Generator().manual_seed(seed)).tolist()
    pool._free = order
    rows = [pool.alloc(h) for h in held]
    before = list(pool._free)
    table_before = [list(r) for r in rows]
    for r, n, h in zip(rows, need, held):
        r.extend(pool.alloc(max(0, n - h)))
    req, pos, slot, start = [], [], [], [0]
    for r, (q, k) in enumerate(zip(q_len, kv_len)):
        for i in range(q):
            req.append(r)
            pos.append(k + i)
            slot.append(rows[r][(k + i) // page] * page + (k + i) % page)
        start.append(start[-1] + q)
    return dict(free=before, table_before=table_before, table=rows, start=start, req=req, pos=pos, slot=slot,
                new_len=[k + q for q, k in zip(q_len, kv_len)], left=pool.n_free)


def prefix_case(groups, H, Hkv, D, page, dtype, seed=0, spread=1.0, positions=None):
    """groups: per group (prefix, [(own keys already there, tokens now), ...] a request).  The rows of a group hold the
    same pages where the prefix fills them; a page that it ends in each row holds for itself."""
    gen = torch.Generator().manual_seed(seed)
    rows, req, pos, start, shared = [], [], [], [0], []
    next_page = 1                                             # (page 0 belongs to nobody: it is NaN)
    copies = []
    for prefix, requests in groups:
        common = list(range(next_page, next_page + prefix // page))
        next_page += len(common)
        first = None
        for own, new in requests:
            n = (prefix + own + new + page - 1) // page - len(common)
            mine = list(range(next_page, next_page + n))
            next_page += n
            if prefix % page and n:
                if first is None:
                    first = mine[0]
                else:
                    copies.append((first, mine[0], prefix % page))
            r = len(rows)
            rows.append((common + mine, prefix + own + new))
            req += [r] * new
            pos += list(range(prefix + own, prefix + own + new))
        start.append(len(req))
        shared.append(prefix)
    width = max(len(r) for r, _ in rows) + 1
    perm = torch.cat([torch.zeros(1, dtype=torch.long), 1 + torch.randperm(next_page - 1, generator=gen)])
    table = torch.zeros(len(rows), width, dtype=torch.int32)
    for i, (r, _) in enumerate(rows):
        table[i, :len(r)] = perm[torch.tensor(r, dtype=torch.long)].int()
    cache = torch.randn(next_page, 2, Hkv, page, D, generator=gen).to(dtype)
    cache[0] = float("nan")
    for a, b, n in copies:
        cache[perm[b], :, :, :n] = cache[perm[a], :, :, :n]
    for r, length in rows:                                    # nothing lies behind a request's last key
        if length % page:
            cache[perm[r[length // page]], :, :, length % page:] = float("nan")
    T = len(req)
    q = (spread * torch.randn(T, H * D, generator=gen)).to(dtype)
    i32 = torch.int32
    return dict(q=q, cache=cache, table=table, req=torch.tensor(req, dtype=i32),
                pos=torch.tensor(pos if positions is None else positions, dtype=i32), start=torch.tensor(start, dtype=i32),
                shared=torch.tensor(shared, dtype=i32), H=H, Hkv=Hkv, D=D, page=page, scale=1.2 / math.sqrt(D))


def prefix_exact(c):
    """(result, sum of p |v|, largest scale * sum |q k|, largest |v|, most keys) in 64 bits."""
    H, Hkv, D, page = c["H"], c["Hkv"], c["D"], c["page"]
    T = c["q"].shape[0]
    out = torch.zeros(T, H * D, dtype=torch.float64)
    mag = torch.zeros(T, H * D, dtype=torch.float64)
    top, vmax, most = 0.0, 0.0, 1
    cache, q = c["cache"].double(), c["q"].double()
    for g in range(len(c["shared"])):
        s = int(c["shared"][g])
        for t in range(int(c["start"][g]), int(c["start"][g + 1])):
            p = int(c["pos"][t])
            if p < 0:
                continue
            lead = c["table"][int(c["req"][int(c["start"][g])])]
            mine = c["table"][int(c["req"][t])]
            at = torch.arange(p + 1)
            pages = torch.where(at < s, lead[at // page], mine[at // page]).long()
            k, v = cache[pages, 0, :, at % page].transpose(0, 1), cache[pages, 1, :, at % page].transpose(0, 1)
            x = q[t].view(Hkv, H // Hkv, D)
            w = torch.softmax(x @ k.transpose(1, 2) * c["scale"], -1)
            out[t] = (w @ v).reshape(-1)
            mag[t] = (w @ v.abs()).reshape(-1)
            top = max(top, float((x.abs() @ k.abs().transpose(1, 2)).max()) * c["scale"])
            vmax, most = max(vmax, float(v.abs().max())), max(most, p + 1)
    return out, mag, top, vmax, most


def prefix_bound(c, exact):
    """How far a result may be off, entry by entry.  A score is a chain of D multiply-adds and two more roundings, each 2^-24
    of at most `top` (D of them as a random walk); its exponential is off by that and by 4 units of 2^-22 / 2 of its own;
    a quotient of sums of them is off by twice that, times the largest value; the sums are n additions, as a random walk.
    bfloat16: the result is rounded (2^-8 of it), and the weights may be before they meet the values (2^-8 of p |v|)."""
    out, mag, top, vmax, most = exact
    u = 2.0 ** -24
    delta = u * top * (math.sqrt(c["D"]) + 3) + 4 * 2 * u
    tol = vmax * (2 * delta + u * (2 * math.sqrt(most) + 8))
    if c["q"].dtype == torch.bfloat16:
        return 2.0 ** -8 * (out.abs() + mag) + tol
    return torch.full_like(out, tol)


def logprobs_exact(logits, tokens, k):
    """(logprob, entropy, place, top ids, top logprobs, bounds) of rows in 64 bits.  NaN in the order as -inf."""
    n, V = logits.shape
    x = logits.double()
    key = torch.where(torch.isnan(x), float("-inf"), x)
    order = torch.sort(key, dim=1, descending=True, stable=True)[1]
    m = x.amax(1, keepdim=True)
    none = (x == float("-inf")).all(1)
    d = x - torch.where(none[:, None], 0.0, m)
    e = torch.exp(d)
    s = e.sum(1, keepdim=True)
    logp = torch.where(none[:, None], float("-inf"), d - torch.log(s))
    dz = torch.where(e > 0, d, 0.0)
    mean = (e * dz).sum(1) / torch.where(none, 1.0, s[:, 0])
    entropy = torch.where(none, 0.0, torch.log(s[:, 0]) - mean)
    asked = (tokens >= 0) & (tokens < V)
    at = tokens.long().clamp(0, V - 1)[:, None]
    place = torch.zeros(n, dtype=torch.int64)
    ranks = torch.empty_like(order).scatter_(1, order, torch.arange(V)[None, :].expand(n, V))
    place = torch.where(asked, ranks.gather(1, at)[:, 0], -1)
    logprob = torch.where(asked, logp.gather(1, at)[:, 0], 0.0)
    # A term of the sum is off by 2 units in the last place of its exponential (2^-22) and by two roundings of its exponent
    # (2^-23 of |l - m|); it enters a chain of at most V / 256 + 32 additions (and joins); then the logarithm and the
    # differences, two roundings each.
    u = 2.0 ** -24
    square = (e * dz * dz).sum(1) / torch.where(none, 1.0, s[:, 0])
    log_s = u * (4 + 2 * mean.abs() + V / 256 + 32 + 2 * torch.log(s[:, 0]).abs())
    tol = log_s[:, None] + u * 4 * (d.abs() + logp.abs())
    tol_entropy = log_s + u * ((4 + V / 256 + 32 + 4) * mean.abs() + 4 * square + 2 * entropy.abs())
    return dict(logprob=logprob, entropy=entropy, place=place, top_ids=order[:, :k], top=logp.gather(1, order[:, :k]),
                tol=tol.gather(1, at)[:, 0], tol_entropy=tol_entropy, tol_top=tol.gather(1, order[:, :k]))
