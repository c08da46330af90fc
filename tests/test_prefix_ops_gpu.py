"""The operators for many requests on one prompt against 64-bit results: lengths from none to long, pages that end inside a
tile, ragged groups, shared heads, rows that see nothing, masked and padded rows, other streams, captured graphs."""
import math

import pytest
import torch

from prefix_cases import logprobs_exact, prefix_bound, prefix_case, prefix_exact, tables_by_hand

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _ops():
    from sglang_c_b200.csrc import ops
    return ops


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


# -- tables ---------------------------------------------------------------------------------------------------------------
def _tables(q_len, kv_len, page, t_cap=None, width=None, seed=0, pad=0):
    """Runs step_tables on what tables_by_hand made; (what it wrote, what it has to be)."""
    want = tables_by_hand(q_len, kv_len, page, seed)
    R, T = len(q_len), len(want["req"])
    width = max([len(r) for r in want["table"]] + [1]) if width is None else width
    whole = torch.full((R + 2, width + 3), -7, dtype=torch.int32, device=DEV)
    for r, row in enumerate(want["table_before"]):
        whole[r, :len(row)] = _i32(row)
    t_cap = T + 3 if t_cap is None else t_cap
    arrays = torch.full((3, t_cap + pad), -9, dtype=torch.int32, device=DEV)
    got = dict(table=whole, q_start=torch.full((R + 2,), -9, dtype=torch.int32, device=DEV), new_len=_i32([-9] * (R + 1)),
               token_req=arrays[0, pad:], positions=arrays[1, pad:], slots=arrays[2, pad:], left=_i32([-9]), status=_i32([-9]))
    return got, want, dict(q_len=_i32(q_len), kv_len=_i32(kv_len), free_pages=_i32(want["free"] + [-3]), n_free=_i32([len(want["free"])]),
                           block_table=whole[:, :width], page_size=page)


def _run_tables(got, args):
    _ops().step_tables(**args, **{k: v for k, v in got.items() if k != "table"})


@pytest.mark.parametrize("q_len,kv_len,page", [
    ([1], [0], 16), ([0], [0], 16), ([0], [33], 16), ([1, 1, 1], [15, 16, 17], 16), ([16, 17, 1], [0, 0, 16], 16), ([5], [3], 1),
    ([3, 0, 0, 7, 0], [0, 5, 0, 9, 64], 8), ([700, 0, 1, 1300], [1, 2, 3, 4], 7), ([4096], [0], 256)])
@pytest.mark.parametrize("pad", [0, 1])
def test_step_tables(q_len, kv_len, page, pad):
    got, want, args = _tables(q_len, kv_len, page, pad=pad)
    _run_tables(got, args)
    _check_tables(got, want)


def _check_tables(got, want):
    R, T = len(want["table"]), len(want["req"])
    assert got["status"].item() == 0 and got["left"].item() == want["left"]
    assert got["q_start"].tolist() == want["start"] + [-9] and got["new_len"].tolist() == want["new_len"] + [-9]
    for name, row in (("token_req", want["req"]), ("positions", want["pos"]), ("slots", want["slot"])):
        assert got[name][:T].tolist() == row and bool((got[name][T:] == -9).all()), name
    for r in range(got["table"].shape[0]):
        row = want["table"][r] if r < R else []
        assert got["table"][r].tolist() == row + [-7] * (got["table"].shape[1] - len(row))


@pytest.mark.parametrize("R,most,context,page", [(64, 1, 900, 16), (513, 40, 200, 16), (5000, 3, 70, 8), (16384, 1, 5, 4), (37, 900, 700, 16)])
def test_step_tables_of_many_requests(R, most, context, page):
    gen = torch.Generator().manual_seed(R)
    q_len = torch.randint(0, most + 1, (R,), generator=gen).tolist()
    kv_len = torch.randint(0, context + 1, (R,), generator=gen).tolist()
    got, want, args = _tables(q_len, kv_len, page, seed=R)
    _run_tables(got, args)
    T = len(want["req"])
    assert got["status"].item() == 0 and got["left"].item() == want["left"]
    for name, row in (("token_req", want["req"]), ("positions", want["pos"]), ("slots", want["slot"])):
        assert torch.equal(got[name][:T].cpu(), torch.tensor(row, dtype=torch.int32)), name
    assert torch.equal(got["q_start"][:R + 1].cpu(), torch.tensor(want["start"], dtype=torch.int32))
    width = got["table"].shape[1]
    table = torch.tensor([r + [-7] * (width - len(r)) for r in want["table"]], dtype=torch.int32)
    assert torch.equal(got["table"][:R].cpu(), table) and bool((got["table"][R:] == -7).all())


@pytest.mark.parametrize("R", [4068, 4069, 4095, 4096])
def test_step_tables_where_shared_memory_needs_an_attribute(R, tmp_path, monkeypatch):
    """About 48 KB of it, in a library loaded afresh: what an earlier call allowed the kernel would hide that this one does not."""
    import ctypes
    import shutil

    from sglang_c_b200.csrc import build
    build.load("step_tables")
    lib = ctypes.CDLL(shutil.copy(build.lib_path("step_tables"), tmp_path / f"tables_{R}.so"))
    lib.sglc_error_string.restype, lib.sglc_error_string.argtypes = ctypes.c_char_p, [ctypes.c_int]
    monkeypatch.setitem(build._loaded, ("step_tables", False), lib)
    got, want, args = _tables([i % 3 for i in range(R)], [i % 50 for i in range(R)], 16)
    _run_tables(got, args)
    T = len(want["req"])
    assert got["status"].item() == 0 and got["left"].item() == want["left"] and got["q_start"].tolist() == want["start"] + [-9]
    for name, row in (("token_req", want["req"]), ("positions", want["pos"]), ("slots", want["slot"])):
        assert got[name].tolist() == row + [-9] * (got[name].numel() - T), name


def test_step_tables_of_no_requests():
    got, want, args = _tables([], [], 16)
    _run_tables(got, args)
    _check_tables(got, want)


@pytest.mark.parametrize("change,status", [
    (dict(n_free=2), 1), (dict(width=2), 2), (dict(t_cap=39), 4), (dict(q_len=[40, -1]), 8), (dict(kv_len=[-1, 0]), 8),
    (dict(n_free=-1), 9), (dict(n_free=10 ** 6), 8), (dict(q_len=[40, 2 ** 31 - 1]), 8), (dict(n_free=2, t_cap=3), 5),
    (dict(q_len=[2 ** 30, 2 ** 30]), 7)])
def test_step_tables_write_all_or_nothing(change, status):
    got, want, args = _tables([40, 0], [0, 0], 16, t_cap=change.get("t_cap"), width=change.get("width"))
    for name in ("q_len", "kv_len"):
        if name in change:
            args[name] = _i32(change[name])
    if "n_free" in change:
        args["n_free"] = _i32([change["n_free"]])
    before = {k: v.clone() for k, v in got.items()}
    _run_tables(got, args)
    assert got["status"].item() == status
    for k, v in got.items():
        assert k == "status" or torch.equal(v, before[k]), k


def test_step_tables_refuse_arrays_that_overlap():
    """Lengths read and written at one word's distance, and an array inside the table; nothing is written."""
    ops = _ops()
    got, want, args = _tables([2, 1, 3], [15, 16, 30], 16)
    x, before = _i32([15, 16, 30, 7, 7]), {k: v.clone() for k, v in got.items()}
    for kw in (dict(args, kv_len=x[:3]), dict(args, q_len=x[:3]), dict(args, free_pages=got["table"].view(-1)[:9])):
        out = {k: v for k, v in got.items() if k != "table"}
        if "kv_len" in kw and kw["kv_len"].data_ptr() == x.data_ptr():
            out["new_len"] = x[1:4]
        if kw["q_len"].data_ptr() == x.data_ptr():
            out["q_start"] = x[1:]
        with pytest.raises(ops.KernelError, match="other memory"):
            ops.step_tables(**kw, **out)
    torch.cuda.synchronize()
    assert x.tolist() == [15, 16, 30, 7, 7] and all(torch.equal(v, before[k]) for k, v in got.items())


def test_step_tables_in_a_graph_follow_the_lengths():
    """A captured call replayed after the lengths, the stack and the table have changed."""
    got, want, args = _tables([1, 2, 3], [15, 16, 30], 16, width=6)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        _run_tables(got, args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        _run_tables(got, args)
    got2, want2, args2 = _tables([2, 0, 4], [16, 33, 1], 16, width=6, seed=5)
    for name in ("q_len", "kv_len", "n_free"):
        args[name].copy_(args2[name])
    args["free_pages"][:len(want2["free"])].copy_(_i32(want2["free"]))
    got["table"].copy_(got2["table"])
    for name in ("q_start", "new_len", "token_req", "positions", "slots"):
        got[name].fill_(-9)
    graph.replay()
    torch.cuda.synchronize()
    _check_tables(got, want2)


# -- attention over shared prefixes ----------------------------------------------------------------------------------------
def _dev(c):
    return {k: v.to(DEV) if torch.is_tensor(v) else v for k, v in c.items()}


def _run_prefix(c, out=None, **kw):
    d = _dev(c)
    out = torch.full(d["q"].shape, 77.0, dtype=d["q"].dtype, device=DEV) if out is None else out
    _ops().attention_prefix(d["q"], d["cache"], d["table"], d["req"], d["pos"], d["start"], d["shared"], out, c["H"], c["scale"], **kw)
    return out


def _check_prefix(c, out, exact=None):
    exact = prefix_exact(c) if exact is None else exact
    first, last = int(c["start"][0]), int(c["start"][-1])
    off = (out.double().cpu() - exact[0]).abs() - prefix_bound(c, exact)
    worst = float(off[first:last].max()) if last > first else -1.0
    assert worst <= 0.0, worst
    assert bool((out[:first] == 77.0).all()) and bool((out[last:] == 77.0).all())
    assert _ops().tc_error_flag(torch.device(DEV)).item() == 0


LAYOUTS = {
    "one token, prefix of one key": [(1, [(0, 1)])],
    "no prefix": [(0, [(0, 1), (40, 1), (3, 2)])],
    "prefix within a page": [(7, [(0, 1), (9, 1)])],
    "ends inside a page and a tile": [(133, [(0, 1), (20, 1), (150, 3)])],
    "whole pages and tiles": [(256, [(0, 1), (16, 1), (1, 1), (31, 1)])],
    "groups of every kind": [(0, [(3, 1)]), (300, [(2, 1)] * 5), (64, []), (17, [(0, 4), (1, 2)]), (129, [(0, 1)])],
    "several tokens a request": [(190, [(0, 37), (5, 20), (70, 1), (0, 64)])],
    "many rows": [(140, [(i % 7, 1 + i % 3) for i in range(70)])],
}


@pytest.mark.parametrize("name", LAYOUTS)
@pytest.mark.parametrize("H,Hkv,D,page", [(2, 2, 64, 16), (8, 2, 128, 64), (5, 1, 64, 8)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_prefix(name, H, Hkv, D, page, dtype):
    c = prefix_case(LAYOUTS[name], H, Hkv, D, page, dtype, seed=len(name) + H)
    _check_prefix(c, _run_prefix(c))


@pytest.mark.parametrize("H,Hkv,D,page", [(3, 3, 8, 16), (4, 2, 40, 5), (6, 1, 72, 16), (2, 1, 96, 48), (12, 3, 136, 3), (4, 4, 192, 32),
                                          (8, 1, 256, 16), (64, 2, 64, 128), (7, 7, 64, 256), (4, 1, 128, 12), (16, 1, 128, 1)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_prefix_heads_and_pages(H, Hkv, D, page, dtype):
    c = prefix_case([(210, [(0, 1), (33, 2), (5, 1)]), (65, [(2, 3)])], H, Hkv, D, page, dtype, seed=D + page)
    _check_prefix(c, _run_prefix(c))


@pytest.mark.parametrize("dtype,H,Hkv,D", [(torch.bfloat16, 12, 12, 64), (torch.bfloat16, 8, 1, 128), (torch.float32, 4, 2, 64)])
@pytest.mark.parametrize("prefix,own", [(6000, 1), (3, 900), (2500, 700)])
def test_attention_prefix_long(dtype, H, Hkv, D, prefix, own):
    """Long prefixes dealt to many blocks, long continuations dealt to clusters; sharp weights."""
    c = prefix_case([(prefix, [(own, 1), (own // 2, 1), (0, 1)])], H, Hkv, D, 16, dtype, seed=prefix, spread=3.0)
    exact = prefix_exact(c)
    for max_own in (1, 256, 5000):
        _check_prefix(c, _run_prefix(c, max_own=max_own), exact)


@pytest.mark.parametrize("H,Hkv,D", [(150, 150, 8), (149, 149, 64), (100, 100, 128), (296, 148, 64)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_prefix_of_whole_items(dtype, H, Hkv, D):
    """About as many items as blocks, of more tiles than one, beside groups without tokens or prefix: blocks take whole items."""
    c = prefix_case([(0, [(3, 1)]), (64, []), (900, [(2, 1)] * 2), (640, []), (1000, [(0, 1), (9, 2)]), (0, [])], H, Hkv, D, 16, dtype, seed=H + D)
    _check_prefix(c, _run_prefix(c))


# (type, key heads, query heads of each, size, tokens a request): those the joining kernel of 16 rows an item takes, and the others
JOINED = [(torch.bfloat16, 2, 4, 64, 1), (torch.bfloat16, 2, 8, 128, 1), (torch.bfloat16, 12, 1, 64, 9), (torch.bfloat16, 8, 1, 128, 9),
          (torch.bfloat16, 3, 5, 64, 9), (torch.bfloat16, 2, 20, 64, 1)]
BY_HEADS = [(torch.bfloat16, 12, 1, 64, 1), (torch.bfloat16, 6, 2, 128, 1), (torch.bfloat16, 4, 4, 40, 1), (torch.float32, 12, 1, 64, 1),
            (torch.float32, 6, 2, 64, 3), (torch.float32, 4, 4, 128, 1)]


def _tokens_where_forms_change(Hkv, gq, tokens, joined):
    """Numbers of tokens just below and from where an item has two warps of its own, and one (by the rules' own constants)."""
    import os
    import re

    from sglang_c_b200.csrc import ops
    here, sms = os.path.dirname(ops.__file__), torch.cuda.get_device_properties(DEV).multi_processor_count

    def constant(name, word):
        with open(os.path.join(here, name)) as f:
            return int(re.search(rf"{word} = (\d+)", f.read()).group(1))
    if joined:
        file, words, each = "attention_prefix_own.cuh", ("JOIN_TWO", "JOIN_ONE"), Hkv * ((gq + 15) // 16)
        of_item = max(n for n in (1, 2, 4, 8, 16) if n == 1 or n * gq <= 16 and n <= tokens)
    else:
        file, words, of_item = "attention_prefix.cu", ("OWN_TWO", "OWN_ONE"), 1
        each = Hkv * gq // (4 if gq % 4 == 0 else 2 if gq % 2 == 0 else 1)
    at = [(-(-constant(file, w) * sms // each) - 1) * of_item + 1 for w in words]          # the first token of the item that does it
    return [(n, form) for a, forms in zip(at, ((4, 2), (2, 1))) for n, form in zip((a - 1, a + 2), forms)]


def _many_tokens(n, dtype, Hkv, gq, D, tokens, seed):
    """n tokens in groups of three kinds, with counts a request about `tokens`; some tokens inside a prefix, one that sees nothing."""
    counts, kinds = [], (1,) if tokens == 1 else (tokens - 2, tokens + 3, tokens, tokens + 1, tokens - 1)
    while sum(counts) < n:
        counts.append(min(kinds[len(counts) % len(kinds)], n - sum(counts)))
    requests = [(i % 7, c) for i, c in enumerate(counts)]
    a, b = len(requests) // 4, len(requests) // 2
    c = prefix_case([(0, requests[:a]), (70, requests[a:b]), (64, []), (33, requests[b:])], Hkv * gq, Hkv, D, 16, dtype, seed=seed)
    second = int(c["start"][1])
    c["pos"][second + 1:second + 4] = torch.tensor([-1, 5, 68])
    return c


@pytest.mark.parametrize("step", range(4))
@pytest.mark.parametrize("kind", JOINED + BY_HEADS)
def test_attention_prefix_of_many_items(kind, step):
    """Enough items that one has two warps, or one, and a block several items, with a last block that is partly empty; results
    on 16 bytes and off them."""
    dtype, Hkv, gq, D, tokens = kind
    n, _ = _tokens_where_forms_change(Hkv, gq, tokens, kind in JOINED)[step]
    c = _many_tokens(n, dtype, Hkv, gq, D, tokens, seed=n + D)
    c["start"][0] = 1
    c["start"][-1] = n - 1
    exact = prefix_exact(c)
    _check_prefix(c, _run_prefix(c), exact)
    wide = torch.full((n, Hkv * gq * D + 11), 77.0, dtype=dtype, device=DEV)
    out = wide[:, 3:3 + Hkv * gq * D]
    _check_prefix(c, _run_prefix(c, out=out), exact)
    assert bool((wide[:, :3] == 77.0).all()) and bool((wide[:, 3 + Hkv * gq * D:] == 77.0).all())


@pytest.mark.parametrize("step", [1, 3])
@pytest.mark.parametrize("kind", [JOINED[0], JOINED[2], JOINED[4], BY_HEADS[0], BY_HEADS[4]])
def test_attention_prefix_of_many_items_with_values_that_are_no_numbers(kind, step):
    """Such a value among each fourth request's own: in the rows that see it, and in none of the others that share its item."""
    dtype, Hkv, gq, D, tokens = kind
    n, _ = _tokens_where_forms_change(Hkv, gq, tokens, kind in JOINED)[step]
    base = _many_tokens(n, dtype, Hkv, gq, D, tokens, seed=n)
    exact = prefix_exact(base)
    c = dict(base, cache=base["cache"].clone())
    sees = torch.zeros(n, dtype=torch.bool)
    group = torch.bucketize(torch.arange(n), base["start"][1:].long(), right=True)
    for r in range(0, len(base["table"]), 4):
        mine = (base["req"] == r).nonzero()[:, 0]
        p = int(base["pos"][mine].max())                      # (its last token's key)
        if p < int(base["shared"][group[mine[0]]]):
            continue
        c["cache"][int(base["table"][r, p // 16]), 1, :, p % 16, 3] = float("nan")
        sees[mine] = base["pos"][mine] >= p
    out = _run_prefix(c).double().cpu()
    off = (out - exact[0]).abs() - prefix_bound(base, exact)
    assert int(sees.sum()) > n // (5 * tokens) and bool((off[~sees] <= 0).all())
    assert not bool(torch.isfinite(out[sees].view(-1, Hkv * gq, D)[..., 3]).any())


@pytest.mark.parametrize("rows", [100, 1024])
@pytest.mark.parametrize("kind", [JOINED[0], JOINED[2], BY_HEADS[3]])
def test_attention_prefix_with_rows_of_the_table_that_no_token_has(kind, rows):
    """A table with a row for every request that a server could hold, in any order; its rows choose the form of the second launch."""
    dtype, Hkv, gq, D, tokens = kind
    c = _many_tokens(40 * tokens, dtype, Hkv, gq, D, tokens, seed=rows)
    where = torch.randperm(rows, generator=torch.Generator().manual_seed(rows))[:len(c["table"])]
    table = torch.full((rows, c["table"].shape[1]), -1, dtype=torch.int32)
    table[where] = c["table"]
    c = dict(c, table=table, req=where[c["req"].long()].int())
    _check_prefix(c, _run_prefix(c))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_prefix_rows_that_see_little(dtype):
    """Tokens inside the prefix see their part of it; one at position -1 sees nothing."""
    pos = [-1, 0, 63, 64, 130, 199, 200, 210]
    c = prefix_case([(200, [(10, 1)] * 8)], 4, 2, 64, 16, dtype, seed=4, positions=pos)
    out = _run_prefix(c)
    _check_prefix(c, out)
    assert bool((out[0] == 0).all())


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("H,Hkv,D", [(2, 2, 64), (8, 2, 128), (4, 4, 136)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_prefix_of_keys_that_are_no_numbers(dtype, H, Hkv, D, which, value):
    """A key (which 0) or value (1) that is no number or infinite, in the prefix and among a request's own: it is in the
    rows that see it and leaves all others as they are."""
    base = prefix_case([(150, [(4, 3), (2, 2), (0, 4), (1, 1)]), (0, [(3, 5)])], H, Hkv, D, 16, dtype, seed=5)
    base["pos"][5:7] = torch.tensor([80, 149])                # (inside the prefix; its last key)
    base["pos"][8] = -1
    exact = prefix_exact(base)
    # (request, position): in the prefix; a request's own; the last position of another; another group's
    for r, p in [(0, 100), (0, 155), (2, 153), (4, 4)]:
        c = dict(base, cache=base["cache"].clone())
        pages = [int(c["table"][r, p // 16])] if p >= 150 or r == 4 else [int(x) for x in c["table"][:4, p // 16].unique()]
        for page in pages:
            c["cache"][page, which, :, p % 16, 5] = value
        sees = (c["pos"] >= p) & ((c["req"] == r) if p >= 150 or r == 4 else (c["req"] < 4))
        out = _run_prefix(c).double().cpu()
        off = (out - exact[0]).abs() - prefix_bound(c, exact)
        assert bool((off[~sees] <= 0).all()), (r, p)
        if which or value != value:                           # (an infinite key may be a weight of 0)
            assert not bool(torch.isfinite(out[sees].view(-1, H, D)[..., 5]).any()), (r, p)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_prefix_strided_rows_and_padded_batches(dtype):
    """Queries and results as columns of wider rows, off 16 bytes; rows before the first group and behind the last one stay."""
    c = prefix_case([(150, [(4, 1)] * 6)], 4, 2, 64, 16, dtype, seed=8)
    exact = prefix_exact(c)
    c["start"] = torch.tensor([2, 5], dtype=torch.int32)
    c["req"][2] = 2
    for shift in (3, 8):
        q = torch.zeros(6, 4 * 64 + 24, dtype=dtype, device=DEV)[:, shift:shift + 256]
        q.copy_(c["q"].to(DEV))
        wide = torch.full((6, 4 * 64 + 24), 77.0, dtype=dtype, device=DEV)
        out = wide[:, shift:shift + 256]
        d = _dev(c)
        _ops().attention_prefix(q, d["cache"], d["table"][:, :30], d["req"], d["pos"], d["start"], d["shared"], out, 4, c["scale"])
        _check_prefix(c, out, exact)
        assert bool((wide[:, :shift] == 77.0).all()) and bool((wide[:, shift + 256:] == 77.0).all())


def test_attention_prefix_without_token_req_and_without_tokens():
    c = prefix_case([(100, [(3, 1), (0, 1)]), (40, [(1, 1)])], 2, 1, 64, 16, torch.bfloat16)
    d = _dev(c)
    out = torch.full_like(d["q"], 77.0)
    _ops().attention_prefix(d["q"], d["cache"], d["table"], None, d["pos"], d["start"], d["shared"], out, 2, c["scale"])
    _check_prefix(c, out)
    none = torch.empty(0, 128, dtype=torch.bfloat16, device=DEV)
    _ops().attention_prefix(none, d["cache"], d["table"], d["req"], d["pos"], d["start"][:1], d["shared"][:0], none, 2, c["scale"])
    keep = torch.full_like(d["q"], 77.0)
    _ops().attention_prefix(d["q"], d["cache"], d["table"], d["req"], d["pos"], _i32([0, 0, 0]), d["shared"], keep, 2, c["scale"])
    assert bool((keep == 77.0).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_prefix_equals_decode_attention(dtype):
    """The same tokens through the attention that reads every request's whole context."""
    c = prefix_case([(500, [(i, 1) for i in range(9)])], 4, 4, 64, 16, dtype, seed=3)
    d = _dev(c)
    d["cache"] = torch.nan_to_num(d["cache"])
    exact = prefix_exact({**c, "cache": d["cache"].cpu()})
    bound = prefix_bound(c, exact)
    out, other = _run_prefix(c), torch.zeros_like(d["q"])
    if dtype == torch.bfloat16:
        _ops().attention_decode(d["q"], d["cache"], d["table"], d["req"], d["pos"], other, 4, c["scale"], None, 512)
    else:
        _ops().attention_simt(d["q"], d["cache"], d["table"], d["req"], d["pos"], other, 4, c["scale"], None, 512, max_q_len=1)
    assert bool(((out.double() - other.double()).abs().cpu() <= 2 * bound).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_prefix_repeats_its_bits(dtype):
    """Twice the same, whatever else ran in the workspace; on another stream; and with a stride of its own."""
    c = prefix_case([(900, [(30, 1)] * 12)], 4, 2, 128, 16, dtype, seed=6)
    first = _run_prefix(c)
    need = _ops().attention_prefix_workspace(12, 1, 4, 2, 128, dtype)
    ws = torch.full((need + 5,), float("nan"), device=DEV)
    assert torch.equal(_run_prefix(c, workspace=ws), first)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = _run_prefix(c)
    torch.cuda.synchronize()
    assert torch.equal(other, first)
    assert bool(torch.isnan(ws[need:]).all())


def test_attention_prefix_on_two_streams_at_once():
    cases = [prefix_case([(2000, [(50 + i, 1)] * 8)], 8, 8, 64, 16, torch.bfloat16, seed=20 + i) for i in range(2)]
    alone = [_run_prefix(c) for c in cases]
    ds = [_dev(c) for c in cases]
    outs = [[torch.zeros_like(d["q"]) for _ in range(20)] for d in ds]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for i in range(20):
        for c, d, o, s in zip(cases, ds, outs, streams):
            with torch.cuda.stream(s):
                _ops().attention_prefix(d["q"], d["cache"], d["table"], d["req"], d["pos"], d["start"], d["shared"], o[i], 8, c["scale"])
    torch.cuda.synchronize()
    for o, a in zip(outs, alone):
        assert all(torch.equal(x, a) for x in o)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_prefix_in_a_graph_follows_the_lengths(dtype):
    """A captured call replayed with other lengths, groups, positions and pages than it was captured with."""
    a = prefix_case([(40, [(3, 1)] * 5), (90, [(1, 1)] * 3)], 4, 2, 64, 16, dtype, seed=1)
    b = prefix_case([(300, [(7, 1)] * 2), (64, [(20, 1)] * 6)], 4, 2, 64, 16, dtype, seed=2)
    n, w = max(a["cache"].shape[0], b["cache"].shape[0]), max(a["table"].shape[1], b["table"].shape[1])
    cache = torch.zeros(n, *a["cache"].shape[1:], dtype=dtype, device=DEV)
    table = torch.zeros(8, w, dtype=torch.int32, device=DEV)
    d = {k: torch.zeros_like(a[k], device=DEV) for k in ("q", "req", "pos", "start", "shared")}
    out = torch.full(a["q"].shape, 77.0, dtype=dtype, device=DEV)

    def fill(c):
        for k in d:
            d[k].copy_(c[k])
        cache[:c["cache"].shape[0]].copy_(c["cache"])
        table[:, :c["table"].shape[1]].copy_(c["table"])

    def call():
        _ops().attention_prefix(d["q"], cache, table, d["req"], d["pos"], d["start"], d["shared"], out, 4, a["scale"])
    fill(a)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        call()
    for c in (b, a, b):
        fill(c)
        out.fill_(77.0)
        graph.replay()
        torch.cuda.synchronize()
        _check_prefix(c, out)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_prefix_does_not_follow_bad_indices(dtype):
    """Pages, requests and positions out of range set the error word and are not read; other tokens' results stand."""
    ops = _ops()
    err = ops.tc_error_flag(torch.device(DEV))
    c = prefix_case([(100, [(20, 1)] * 4), (64, [(5, 1)] * 3)], 4, 2, 64, 16, dtype, seed=12)
    good = _run_prefix(c)
    bad = {k: v.clone() if torch.is_tensor(v) else v for k, v in c.items()}
    bad["table"][1, 7] = c["cache"].shape[0]            # a page of token 1's own keys
    bad["table"][2, 7] = -5
    bad["req"][3] = 99
    bad["pos"][5] = 10 ** 6
    bad["table"][4:, 2] = 1 << 30                       # (a page of the second group's prefix, in all of its rows)
    out = _run_prefix(bad)
    torch.cuda.synchronize()
    assert err.item() & 4
    err.zero_()
    assert torch.equal(out[0], good[0])
    starts = _run_prefix({**c, "start": torch.tensor([0, 6, 2, 7], dtype=torch.int32), "shared": torch.tensor([100, 64, 90], dtype=torch.int32)})
    torch.cuda.synchronize()
    err.zero_()
    exact = prefix_exact(c)
    assert bool(((starts[0].double().cpu() - exact[0][0]).abs() <= prefix_bound(c, exact)[0]).all())
    starts = _run_prefix({**c, "start": torch.tensor([-4, 4, 900], dtype=torch.int32)})
    torch.cuda.synchronize()
    assert torch.equal(starts[:4], good[:4]) and err.item() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_prefix_beside_its_bounds_check_build(dtype):
    """Both builds' libraries in one process, each with state of its own."""
    from sglang_c_b200.csrc import build
    c = prefix_case([(300, [(9, 1)] * 5)], 4, 2, 64, 16, dtype, seed=9)
    first = _run_prefix(c)
    build.set_bounds_check(True)
    try:
        assert torch.equal(_run_prefix(c), first)
    finally:
        build.set_bounds_check(False)
    assert torch.equal(_run_prefix(c), first)


def test_attention_prefix_beyond_32_bits():
    """Pages whose offset in the cache passes 2^31 and 2^32 elements."""
    n_pages, page, Hkv, D = 70000, 64, 4, 128
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 10 GB")
    cache = torch.zeros(n_pages, 2, Hkv, page, D, dtype=torch.bfloat16, device=DEV)
    c = prefix_case([(300, [(40, 1)] * 3)], 8, Hkv, D, page, torch.bfloat16, seed=2)
    small = _run_prefix(c)
    far = n_pages - 1 - 3001 * torch.arange(c["cache"].shape[0])
    cache[far.to(DEV)] = c["cache"].to(DEV)
    d = _dev({**c, "table": far[c["table"].long()].int()})
    out = torch.zeros_like(d["q"])
    _ops().attention_prefix(d["q"], cache, d["table"], d["req"], d["pos"], d["start"], d["shared"], out, 8, c["scale"])
    assert torch.equal(out, small)


# -- log-probabilities -----------------------------------------------------------------------------------------------------
def _logprobs(x, tokens, k, top_pad=0):
    n = x.shape[0]
    f = dict(dtype=torch.float32, device=DEV)
    got = dict(logprob=torch.full((n,), 7.0, **f), entropy=torch.full((n,), 7.0, **f), place=_i32([7] * n),
               top_ids=torch.full((n, k + top_pad), 7, dtype=torch.int32, device=DEV)[:, :k],
               top_logprobs=torch.full((n, k + top_pad), 7.0, **f)[:, :k])
    _ops().token_logprobs(x, tokens, got["logprob"], entropy=got["entropy"], place=got["place"], top_ids=got["top_ids"],
                          top_logprobs=got["top_logprobs"])
    return {a: b.cpu() for a, b in got.items()}


def _near(x, y, tol):
    x, y = x.double(), y.double()
    # (results are float32: a difference of two of its largest numbers, -5.6e38, lies below -3.4e38 and rounds to -inf)
    y = torch.where(y.abs() > torch.finfo(torch.float32).max, torch.sign(y) * math.inf, y)
    same = (x == y) | (torch.isnan(x) & torch.isnan(y)) | ((x - y).abs() <= tol)
    assert bool(same.all()), (x[~same][:5], y[~same][:5])


def _check_logprobs(x, tokens, k, got):
    want = logprobs_exact(x.cpu(), tokens.cpu(), k)
    assert torch.equal(got["place"].long(), want["place"])
    assert torch.equal(got["top_ids"].long(), want["top_ids"])
    _near(got["logprob"], want["logprob"], want["tol"])
    _near(got["entropy"], want["entropy"], want["tol_entropy"])
    _near(got["top_logprobs"], want["top"], want["tol_top"])


@pytest.mark.parametrize("n,V", [(1, 1), (3, 2), (1, 50257), (2, 333), (5, 1024), (64, 4099), (7, 50257), (300, 777), (600, 5000), (1, 300001),
                                 (40, 70001)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("k", [0, 1, 5, 64])
def test_token_logprobs(n, V, dtype, k):
    k = min(k, V)
    gen = torch.Generator(device=DEV).manual_seed(n + V)
    x = (4 * torch.randn(n, V, generator=gen, device=DEV)).to(dtype)
    tokens = torch.randint(0, V, (n,), generator=gen, device=DEV, dtype=torch.int32)
    tokens[::3] = x[::3].float().argmax(1).int()
    _check_logprobs(x, tokens, k, _logprobs(x, tokens, k))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shift,pad", [(0, 1), (1, 0), (3, 6), (5, 3), (7, 9)])
def test_token_logprobs_rows_off_16_bytes_between_what_is_no_number(dtype, shift, pad):
    wide = torch.full((11, shift + 2001 + pad), float("nan"), dtype=dtype, device=DEV)
    x = wide[:, shift:shift + 2001]
    x.copy_(torch.randn(11, 2001, generator=torch.Generator(device=DEV).manual_seed(shift), device=DEV))
    tokens = _i32([0, 1, 2, 3, 1997, 1998, 1999, 2000, 5, 6, 7])
    _check_logprobs(x, tokens, 9, _logprobs(x, tokens, 9, top_pad=2))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 40, 700])
def test_token_logprobs_ties_go_to_the_lowest_id(dtype, n):
    """All logits one number, few numbers, a thread's whole stride of large ones, and ascending or descending rows."""
    V = 9001
    at = torch.arange(V, device=DEV)
    gen = torch.Generator(device=DEV).manual_seed(n)
    few = torch.randint(0, 3, (V,), generator=gen, device=DEV).float()
    rows = [torch.zeros(V, device=DEV), few, (at % 1024 < 8).float() * 3 + (at % 7).float() * 0.25, (at % 2048 // 8 == 3).float() * 5,
            at.float() * 2.0 ** -6, -at.float() * 2.0 ** -6, (at == V - 1).float(), -0.0 * (at % 2).float(),
            (at % 4096 < 16).float() * at.float() * 2.0 ** -6]
    x = torch.stack([rows[i % len(rows)] for i in range(n)]).to(dtype) if n > 1 else None
    if n == 1:
        for r in rows:
            for k in (1, 20, 64):
                t = _i32([V // 2])
                _check_logprobs(r[None].to(dtype), t, k, _logprobs(r[None].to(dtype), t, k))
        return
    tokens = torch.randint(0, V, (n,), generator=gen, device=DEV, dtype=torch.int32)
    for k in (20, 64):
        _check_logprobs(x, tokens, k, _logprobs(x, tokens, k))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [8, 900])
def test_token_logprobs_masked_rows(dtype, n):
    """Few allowed tokens, fewer than the alternatives asked for, one, none; masks of the type's lowest value; tokens that are
    not allowed; rows that ask for none."""
    V, low = 5003, torch.finfo(dtype).min
    gen = torch.Generator(device=DEV).manual_seed(n)
    x = (3 * torch.randn(n, V, generator=gen, device=DEV)).to(dtype)
    keep = torch.zeros(n, V, dtype=torch.bool, device=DEV)
    for r in range(n):
        many = (0, 1, 3, 10, 50, 2000, 5003)[r % 7]
        keep[r, torch.randperm(V, generator=gen, device=DEV)[:many]] = True
    tokens = torch.randint(0, V, (n,), generator=gen, device=DEV, dtype=torch.int32)
    tokens[3::5] = x.masked_fill(~keep, float("-inf")).float().argmax(1).int()[3::5]
    tokens[4::7] = -1
    tokens[5::11] = V
    tokens[6::13] = 2 ** 31 - 1
    for fill in (float("-inf"), low):
        y = x.masked_fill(~keep, fill)
        _check_logprobs(y, tokens, 20, _logprobs(y, tokens, 20))


@pytest.mark.parametrize("n", [1, 600])
def test_token_logprobs_of_what_is_no_number(n):
    """NaN and +inf make a row's log-probabilities and entropy NaN and leave the order as it is (NaN last); numbers of any size."""
    V = 3001
    x = torch.randn(n + 8, V, generator=torch.Generator(device=DEV).manual_seed(n), device=DEV)
    x[0, 5] = float("nan")
    x[1, 6] = float("inf")
    x[2] = float("nan")
    x[3, ::2] = float("nan")
    x[3, 1::2] = float("-inf")
    x[4] *= 1e38
    x[5] = x[5] * 1e-3 + 3e38
    x[6, 3:] = float("-inf")
    x[6, 1] = float("nan")
    x[7] *= 1e-40
    tokens = torch.randint(0, V, (n + 8,), generator=torch.Generator(device=DEV).manual_seed(7), device=DEV, dtype=torch.int32)
    if n == 1:
        for r in range(9):
            _check_logprobs(x[r:r + 1], tokens[r:r + 1], 12, _logprobs(x[r:r + 1], tokens[r:r + 1], 12))
    else:
        _check_logprobs(x, tokens, 12, _logprobs(x, tokens, 12))


def test_token_logprobs_gives_what_is_asked():
    """Each output alone, no rows at all, and tokens None."""
    ops = _ops()
    x = torch.randn(5, 400, device=DEV)
    tokens = _i32([1, 2, 3, 4, 5])
    whole = _logprobs(x, tokens, 3)
    lp = torch.zeros(5, device=DEV)
    ops.token_logprobs(x, tokens, lp)
    assert torch.equal(lp.cpu(), whole["logprob"])
    h = torch.zeros(5, device=DEV)
    ops.token_logprobs(x, None, lp, entropy=h)
    assert torch.equal(h.cpu(), whole["entropy"]) and bool((lp == 0).all())
    ops.token_logprobs(x[:0], tokens[:0], lp[:0])
    ops.token_logprobs(x, tokens, lp, top_ids=torch.zeros(5, 0, dtype=torch.int32, device=DEV), top_logprobs=torch.zeros(5, 0, device=DEV))
    assert torch.equal(lp.cpu(), whole["logprob"])


def test_token_logprobs_beyond_32_bits():
    """Rows whose offset passes 2^31 elements."""
    V, n = 200003, 11000
    if torch.cuda.mem_get_info()[0] < 6 << 30:
        pytest.skip("needs 5 GB")
    x = torch.zeros(n, V, dtype=torch.bfloat16, device=DEV)
    x[-3:] = torch.randn(3, V, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV)
    tokens = torch.arange(n, device=DEV, dtype=torch.int32)
    got = _logprobs(x, tokens, 4)
    _check_logprobs(x[-3:], tokens[-3:], 4, {k: v[-3:] for k, v in got.items()})


# -- together --------------------------------------------------------------------------------------------------------------
def test_many_answers_to_one_prompt():
    """A loop as a server makes it, on the device alone: the step's arrays from the lengths, the new keys and values into their
    slots, attention over the shared prompt, a head, log-probabilities of the tokens taken; one captured graph a parity of the
    step (the lengths go back and forth between two buffers), against the same in 64 bits from the tables of the host's pool."""
    ops = _ops()
    N, H, Hkv, D, page, prompt, V, steps = 7, 4, 2, 64, 16, 150, 321, 20
    gen = torch.Generator().manual_seed(5)

    def rand(*shape):
        return torch.randn(shape, generator=gen)
    n_pages = 60
    shared_pages = prompt // page
    order = torch.randperm(n_pages, generator=gen).tolist()
    cache = rand(n_pages, 2, Hkv, page, D).bfloat16()
    # the prompt's last, partly filled page is each answer's own
    table = torch.zeros(N, 20, dtype=torch.int32)
    common, rest = order[:shared_pages], order[shared_pages:]
    for r in range(N):
        mine = rest.pop()
        table[r, :shared_pages + 1] = torch.tensor(common + [mine])
        cache[mine, :, :, :prompt % page] = cache[table[0, shared_pages], :, :, :prompt % page]
    d_cache, d_table = cache.to(DEV), table.to(DEV)
    free = _i32(rest)
    counts, lens = [_i32([len(rest)]), _i32([0])], [_i32([prompt] * N), _i32([0] * N)]
    q_len, status = _i32([1] * N), _i32([0])
    arrays = {k: torch.zeros(N, dtype=torch.int32, device=DEV) for k in ("token_req", "positions", "slots")}
    q_start = torch.zeros(N + 1, dtype=torch.int32, device=DEV)
    group, shared = _i32([0, N]), _i32([prompt])
    qkv = rand(steps, N, (H + 2 * Hkv) * D).bfloat16()
    w = (rand(V, H * D) * 0.05).bfloat16()
    tokens = torch.randint(0, V, (steps, N), generator=gen, dtype=torch.int32)
    d_qkv, d_tok = torch.zeros(N, (H + 2 * Hkv) * D, dtype=torch.bfloat16, device=DEV), torch.zeros(N, dtype=torch.int32, device=DEV)
    d_w, out = w.to(DEV), torch.zeros(N, H * D, dtype=torch.bfloat16, device=DEV)
    logits = torch.zeros(N, V, device=DEV)
    lp, place, ids, top = torch.zeros(N, device=DEV), _i32([0] * N), torch.zeros(N, 5, dtype=torch.int32, device=DEV), torch.zeros(N, 5, device=DEV)

    def step(i):
        a, b = i % 2, 1 - i % 2
        ops.step_tables(q_len, lens[a], free, counts[a], d_table, page, q_start, lens[b], arrays["token_req"], arrays["positions"],
                        arrays["slots"], counts[b], status)
        ops.kv_write(d_qkv[:, H * D:(H + Hkv) * D], d_qkv[:, (H + Hkv) * D:], d_cache, arrays["slots"], Hkv, D)
        ops.attention_prefix(d_qkv[:, :H * D], d_cache, d_table, arrays["token_req"], arrays["positions"], group, shared, out, H,
                             0.125, max_own=steps)
        ops.gemm_simt(out, d_w, None, out=logits)
        ops.token_logprobs(logits, d_tok, lp, place=place, top_ids=ids, top_logprobs=top)

    graphs = {}
    saved = [t.clone() for t in (*counts, *lens, d_table, d_cache)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(0)
    torch.cuda.synchronize()
    for i in (0, 1):
        graphs[i] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graphs[i], stream=s):
            step(i)
    for t, v in zip((*counts, *lens, d_table, d_cache), saved):
        t.copy_(v)
    ref_cache, ref_table, pool = cache.clone(), table.clone(), list(rest)
    for i in range(steps):
        d_qkv.copy_(qkv[i])
        d_tok.copy_(tokens[i])
        torch.cuda.synchronize()
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        p = prompt + i
        for r in range(N):
            if p % page == 0:
                ref_table[r, p // page] = pool.pop()
            at = ref_table[r, p // page].item()
            ref_cache[at, 0, :, p % page] = qkv[i, r, H * D:(H + Hkv) * D].view(Hkv, D)
            ref_cache[at, 1, :, p % page] = qkv[i, r, (H + Hkv) * D:].view(Hkv, D)
        c = dict(q=qkv[i][:, :H * D], cache=ref_cache, table=ref_table, req=torch.arange(N), pos=torch.full((N,), p), start=[0, N],
                 shared=[prompt], H=H, Hkv=Hkv, D=D, page=page, scale=0.125)
        exact = prefix_exact(c)
        assert status.item() == 0 and torch.equal(d_table.cpu(), ref_table) and counts[1 - i % 2].item() == len(pool)
        assert bool(((out.double().cpu() - exact[0]).abs() <= prefix_bound(c, exact)).all())
        got = dict(logprob=lp.cpu(), place=place.cpu(), top_ids=ids.cpu(), top_logprobs=top.cpu())
        want = logprobs_exact(logits.cpu(), tokens[i], 5)
        assert torch.equal(got["place"].long(), want["place"]) and torch.equal(got["top_ids"].long(), want["top_ids"])
        _near(got["logprob"], want["logprob"], want["tol"])
        _near(got["top_logprobs"], want["top"], want["tol_top"])
        assert math.isfinite(float(lp.sum()))
