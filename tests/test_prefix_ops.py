"""The operators for many requests on one prompt, without a GPU: what their entry points refuse."""
import pytest
import torch

from sglang_c_b200.csrc import build, ops


@pytest.fixture
def host(monkeypatch):
    """The entry points' checks on tensors of the host; a call that passes them all ends in `Launched`."""
    class Launched(Exception):
        pass

    def function(library, name, types, result=None):
        def sizes(T, G, H, Hkv, D, dt):
            assert len(types) == 6
            return 1000 if H % Hkv == 0 and D % 8 == 0 and D <= 256 and G <= ops.PREFIX_GROUPS else -1

        def launch(*args):
            assert len(args) == len(types)
            for a, t in zip(args, types):
                assert isinstance(a, float if t == "f" else (int, type(None)) if t == "p" else int), (name, t, a)
            raise Launched
        return None, sizes if name == "sglc_attention_prefix_workspace" else launch

    monkeypatch.setattr(ops, "_here", lambda what, *t: 0)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(ops, "_prefix_sizes", {})
    monkeypatch.setattr(ops, "_stream_here", lambda device: 0)
    monkeypatch.setattr(ops, "tc_error_flag", lambda device: torch.zeros(1, dtype=torch.int32))
    monkeypatch.setattr(ops, "_function", function)
    return Launched


def _i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def _tables(**kw):
    a = dict(q_len=_i32(3), kv_len=_i32(3), free_pages=_i32(9), n_free=_i32(1), block_table=_i32(4, 6), page_size=16, q_start=_i32(4),
             new_len=_i32(3), token_req=_i32(20), positions=_i32(20), slots=_i32(20), left=_i32(1), status=_i32(1))
    a.update(kw)
    ops.step_tables(**a)


_same = _i32(3)


@pytest.mark.parametrize("kw,words", [
    (dict(q_len=torch.zeros(3)), "q_len must be a contiguous int32"), (dict(slots=_i32(40)[::2]), "slots must be a contiguous"),
    (dict(block_table=_i32(2, 6)), "rows for 3 requests"), (dict(block_table=_i32(6, 4).t()), "rows for 3 requests"),
    (dict(block_table=_i32(1, 6).expand(4, 6)), "rows for 3 requests"), (dict(block_table=_i32(24)), "rows for 3 requests"),
    (dict(q_start=_i32(3)), "one more"), (dict(kv_len=_i32(2)), "an entry a request"), (dict(slots=_i32(19)), "one length"),
    (dict(n_free=_i32(0)), "one word each"), (dict(page_size=0), "page size 0"), (dict(page_size=1 << 21), "page size"),
    (dict(q_len=_i32(20000)), "at most 16384"), (dict(kv_len=_same, new_len=_same), "other memory")])
def test_step_tables_refuses(host, kw, words):
    with pytest.raises(host):
        _tables()
    with pytest.raises(ops.KernelError, match=words):
        _tables(**kw)


def test_step_tables_refuses_one_word_for_both_counts(host):
    n = _i32(1)
    with pytest.raises(ops.KernelError, match="other memory"):
        _tables(n_free=n, left=n)


def test_step_tables_refuses_what_it_reads_as_what_it_writes(host):
    x, words, tokens = _i32(20), _i32(2), _i32(20)
    for kw in (dict(q_len=x[:3], q_start=x[:4]), dict(n_free=words[:1], status=words[:1]), dict(left=words[:1], status=words[:1]),
               dict(kv_len=tokens[:3], positions=tokens), dict(slots=tokens, positions=tokens)):
        with pytest.raises(ops.KernelError, match="other memory"):
            _tables(**kw)
    none = _i32(0)
    with pytest.raises(host):                              # (arrays without entries are no memory)
        _tables(q_len=none, kv_len=none, new_len=none, token_req=none, positions=none, slots=none)
    with pytest.raises(host):                              # (what is only read may be one array)
        _tables(q_len=x[:3], kv_len=x[:3])


_SPANS = dict(q_len=(0, 5), kv_len=(10, 5), free_pages=(20, 9), n_free=(30, 1), table=(100, 0), q_start=(40, 6), new_len=(50, 5),
              token_req=(60, 8), positions=(70, 8), slots=(80, 8), left=(90, 1), status=(92, 1))


def _overlap(stride=7, width=4, R=5, **at):
    """The launcher's look at arrays at made-up addresses (words from 2^20 on; nothing is read)."""
    import ctypes
    p = {k: ctypes.c_void_p((1 << 20) + 4 * at.get(k, v[0])) for k, v in _SPANS.items()}
    return build.load("step_tables").sglc_step_tables_overlap(
        p["q_len"], p["kv_len"], p["free_pages"], 9, p["n_free"], p["table"], ctypes.c_longlong(stride), width, R, p["q_start"],
        p["new_len"], p["token_req"], p["positions"], p["slots"], 8, p["left"], p["status"])


_READ = ("q_len", "kv_len", "free_pages", "n_free")


def test_step_tables_overlaps_word_by_word():
    """Every written array against every other one: overlap by a word at either end, and side by side."""
    assert _overlap() == 0
    names = [n for n in _SPANS if n != "table"]
    for a in names:
        for b in names:
            if a == b:
                continue
            far = {a: 1000}                                  # (a clear of the rest, b moved along it)
            size_a, size_b = _SPANS[a][1], _SPANS[b][1]
            for start in (1000 - size_b, 1000 - size_b + 1, 1000, 1000 + size_a - 1, 1000 + size_a):
                meets = start + size_b > 1000 and start < 1000 + size_a
                want = int(meets and not (a in _READ and b in _READ))
                assert _overlap(**far, **{b: start}) == want, (a, b, start)


def test_step_tables_overlaps_with_the_table():
    """An array in one of the table's rows, each word of it; between rows (7 words apart, 4 of them the row's) there is room for one."""
    inside = {100 + 7 * r + i for r in range(5) for i in range(4)}
    for name, (_, size) in _SPANS.items():
        if name == "table":
            continue
        for start in range(85, 150):
            want = int(any(w in inside for w in range(start, start + size)))
            others = {n: 2000 + 50 * i for i, n in enumerate(_SPANS) if n not in (name, "table")}
            assert _overlap(**{**others, name: start}) == want, (name, start)
    assert _overlap(R=0, table=40) == 0 and _overlap(width=0, table=50) == 0        # (no rows, or rows without entries)


def _prefix(**kw):
    a = dict(q=torch.zeros(5, 48), cache=torch.zeros(7, 2, 2, 4, 8), block_table=_i32(3, 4), token_req=_i32(5), positions=_i32(5),
             group_start=_i32(3), shared_len=_i32(2), out=torch.zeros(5, 48), n_heads=6, scale=0.3)
    a.update(kw)
    ops.attention_prefix(**a)


@pytest.mark.parametrize("kw,words", [
    (dict(q=torch.zeros(5, 40)), "do not match heads"), (dict(out=torch.zeros(4, 48)), "do not match heads"),
    (dict(q=torch.zeros(48, 5).t()), "do not match heads"), (dict(out=torch.zeros(1, 48).expand(5, 48)), "rows of out overlap"),
    (dict(q=torch.zeros(5, 48).bfloat16()), "one dtype"), (dict(out=torch.zeros(5, 48).half()), "one dtype"),
    (dict(cache=torch.zeros(7, 1, 2, 4, 8)), "the cache is"), (dict(cache=torch.zeros(7, 2, 2, 4, 16)[..., ::2]), "the cache is"),
    (dict(cache=torch.zeros(7 * 128 + 1)[1:].view(7, 2, 2, 4, 8)), "begin on 16 bytes"),
    (dict(block_table=torch.zeros(3, 4)), "int32 rows"), (dict(block_table=_i32(4, 3).t()), "int32 rows"),
    (dict(positions=_i32(4)), "an entry a token"), (dict(token_req=_i32(4)), "an entry a token"),
    (dict(group_start=_i32(2)), "one more than"), (dict(positions=torch.zeros(5)), "positions must be"),
    (dict(scale=0.0), "must be positive"), (dict(scale=float("nan")), "must be positive"), (dict(scale=float("inf")), "must be positive"),
    (dict(workspace=torch.zeros(999)), "1000 float32"), (dict(workspace=torch.zeros(2000)[::2]), "1000 float32"),
    (dict(q=torch.zeros(5, 40), out=torch.zeros(5, 40), n_heads=5), "whole groups"),
    (dict(group_start=_i32(258), shared_len=_i32(257)), "at most 256 groups")])
def test_attention_prefix_refuses(host, kw, words):
    with pytest.raises(host):
        _prefix()
    with pytest.raises(ops.KernelError, match=words):
        _prefix(**kw)


def test_attention_prefix_refuses_other_types_and_sizes(host):
    half = torch.float16
    with pytest.raises(ops.KernelError, match="is not handled"):
        _prefix(q=torch.zeros(5, 48, dtype=half), out=torch.zeros(5, 48, dtype=half), cache=torch.zeros(7, 2, 2, 4, 8, dtype=half))
    with pytest.raises(ops.KernelError, match="multiples of 8 up to 256"):
        _prefix(q=torch.zeros(5, 72), out=torch.zeros(5, 72), cache=torch.zeros(7, 2, 2, 4, 12))
    with pytest.raises(ops.KernelError, match="multiples of 8 up to 256"):
        _prefix(q=torch.zeros(5, 6 * 264), out=torch.zeros(5, 6 * 264), cache=torch.zeros(7, 2, 2, 4, 264))


def _logprobs(**kw):
    a = dict(logits=torch.zeros(4, 100), tokens=_i32(4), logprob=torch.zeros(4), entropy=torch.zeros(4), place=_i32(4),
             top_ids=_i32(4, 3), top_logprobs=torch.zeros(4, 3))
    a.update(kw)
    ops.token_logprobs(**a)


@pytest.mark.parametrize("kw,words", [
    (dict(logits=torch.zeros(4, 100).half()), "is not handled"), (dict(logits=torch.zeros(100, 4).t()), "rows of a vocabulary"),
    (dict(logits=torch.zeros(400)), "rows of a vocabulary"), (dict(logits=torch.zeros(4, 0)), "rows of a vocabulary"),
    (dict(tokens=torch.zeros(4, dtype=torch.int64)), "tokens must be"), (dict(tokens=_i32(5)), "tokens must be"),
    (dict(logprob=torch.zeros(4).double()), "logprob must be"), (dict(logprob=torch.zeros(8)[::2]), "logprob must be"),
    (dict(entropy=torch.zeros(3)), "entropy must be"), (dict(place=torch.zeros(4)), "place must be"),
    (dict(top_logprobs=None), "come together"), (dict(top_ids=None), "come together"),
    (dict(top_ids=_i32(4, 2)), r"\[rows, k\] both"), (dict(top_ids=torch.zeros(4, 3)), r"\[rows, k\] both"),
    (dict(top_ids=_i32(4, 65), top_logprobs=torch.zeros(4, 65)), "at most 64"),
    (dict(logits=torch.zeros(4, 2)), "3 alternatives of 2"),
    (dict(top_ids=_i32(4, 6)[:, ::2], top_logprobs=torch.zeros(4, 6)[:, ::2]), "one stride"),
    (dict(top_ids=_i32(4, 5)[:, :3]), "one stride"),
    (dict(top_ids=_i32(1, 3).expand(4, 3), top_logprobs=torch.zeros(1, 3).expand(4, 3)), "overlap")])
def test_token_logprobs_refuses(host, kw, words):
    with pytest.raises(host):
        _logprobs()
    with pytest.raises(host):
        _logprobs(tokens=None, entropy=None, place=None, top_ids=None, top_logprobs=None)
    with pytest.raises(ops.KernelError, match=words):
        _logprobs(**kw)


def test_they_refuse_tensors_of_the_host(monkeypatch):
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    for call in (_tables, _prefix, _logprobs):
        with pytest.raises(ops.KernelError, match="CUDA tensors only"):
            call()


def test_they_refuse_tensors_of_another_device(monkeypatch):
    """Tensors of device 1 while device 0 is current: the kernels would run on the wrong one's stream."""
    class There:
        device, is_cuda = "cuda:1", True

        def get_device(self):
            return 1
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    assert ops._here("x", None) == 0
    with pytest.raises(ops.KernelError, match="lies on cuda:1, the current device is cuda:0"):
        ops._here("x", None, There())


def test_sizes_beyond_32_bits_are_refused(host):
    """(Tensors of torch's device without memory.)"""
    for shape in ((4, 1 << 30), (1 << 30, 1)):
        logits = torch.empty(shape, device="meta")
        with pytest.raises(ops.KernelError, match="at most 536870912 both"):
            _logprobs(logits=logits)
    with pytest.raises(ops.KernelError, match="at most 536870912"):
        _prefix(q=torch.empty((1 << 30, 48), device="meta"))
    with pytest.raises(ops.KernelError, match="100000000 tokens of 6 heads .at most 536870912"):
        _prefix(q=torch.empty((100000000, 48), device="meta"))
    with pytest.raises(ops.KernelError, match="at most 16384 and 536870912"):
        _tables(token_req=torch.empty(1 << 30, dtype=torch.int32, device="meta"))
    with pytest.raises(ops.KernelError, match="a cache of 0 pages"):
        _prefix(cache=torch.zeros(0, 2, 2, 4, 8))


def test_the_sizes_named_here_are_the_kernels():
    """What the bindings say of limits is what the sources say."""
    import os
    import re
    here = os.path.dirname(ops.__file__)

    def constant(name, word):
        with open(os.path.join(here, name)) as f:
            return int(re.search(rf"constexpr int {word} = (\d+)", f.read()).group(1))
    assert constant("step_tables.cu", "MAX_REQUESTS") == ops.STEP_TABLES_REQUESTS
    assert constant("attention_prefix.cuh", "MAX_GROUPS") == ops.PREFIX_GROUPS
    assert constant("token_logprobs.cu", "MAX_TOP") == ops.TOP_TOKENS
