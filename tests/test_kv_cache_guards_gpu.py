"""4-bit key/value cache on the GPU at the edge of what is allowed.  Bounds as
in test_kv_cache_gpu.py, whose cases these use."""
import threading

import numpy as np
import pytest
import torch

import kv4_oracle as ko
from test_kv_cache_gpu import (TINY, U, Case, _device, append_reference, device_error, f64,  # noqa: F401 (a fixture)
                               places)

pytestmark = pytest.mark.gpu


def check_seen(case, q, out, log_sum, seen, scale=None):
    """Row t of the step against the oracle on the tokens `seen[t]` = (sequence,
    indices) that it sees."""
    scale = q.shape[2] ** -0.5 if scale is None else scale
    held = [(case.sequence(b, 0), case.sequence(b, 1)) for b in range(len(case.lengths))]
    got, lse = f64(out), f64(log_sum)
    for t, (b, idx) in enumerate(seen):
        k, v = (x[idx] for x in held[b])
        ref, want, spread, size, mass = (x[0] for x in ko.attention(f64(q[t:t + 1]), k, v, scale, 1, causal=False))
        d = 2.0**-16 * size
        tol = (np.maximum(U[out.dtype] * np.abs(ref), TINY[out.dtype]) + (2.0**-11 + 2 * d[:, None]) * spread
               + 2.0**-31 * mass + 1e-30)
        assert (np.abs(got[t] - ref) <= tol).all(), t
        if len(idx):
            assert (np.abs(lse[t] - want) <= d + 2.0**-20 * (1 + np.abs(want))).all(), t
        else:
            assert not got[t].any() and (lse[t] == -np.inf).all(), t


def test_threads_share_a_batch_and_a_stream():
    """Calls of several host threads on their common default stream, each with
    parts to join: every thread gets the bits of its own call."""
    case = Case([2100, 900], [1, 1], 2, 128, page=32, junk=True)
    queries = [case.queries(8, 128, torch.float16) for _ in range(4)]
    want = [case.cache.attention(q, case.batch) for q in queries]
    for q, y in zip(queries, want):
        case.check(q, y)
    got = [[] for _ in queries]
    go = threading.Barrier(len(queries))

    def calls(i):
        go.wait(30)
        got[i] += [case.cache.attention(queries[i], case.batch) for _ in range(50)]

    threads = [threading.Thread(target=calls, args=(i,)) for i in range(len(queries))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for ys, y in zip(got, want):
        assert len(ys) == 50 and all(torch.equal(x, y) for x in ys)
    assert device_error() == 0


def test_two_streams_in_flight_at_once():
    case = Case([3000, 500, 1200], [1, 1, 1], 2, 64, page=16, junk=True)
    q = [case.queries(16, 64, torch.bfloat16) for _ in range(2)]
    want = [case.cache.attention(x, case.batch) for x in q]
    case.check(q[0], want[0])
    case.check(q[1], want[1])
    streams = [torch.cuda.Stream() for _ in q]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(40):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(case.cache.attention(q[i], case.batch))
    torch.cuda.synchronize()
    for ys, y in zip(got, want):
        assert all(torch.equal(x, y) for x in ys)


@pytest.mark.parametrize("length, count, kept", [(33, 1, []), (33, 2, [0]), (34, 5, [0, 1, 2]), (1 << 30, 2, []),
                                                 ((1 << 31) - 1, 3, []), (1, 3, [2]), (-5, 2, []),
                                                 (-(1 << 31), 3, [])])
def test_append_beyond_the_page_table(length, count, kept):
    """Tokens whose place is outside the page table (of 32 here) are left out
    with an error: none of them lands on a token that is there."""
    from openquant_b200.kv_cache import Int4KVCache, KVBatch, rotary_table

    dev = dict(dtype=torch.int32, device="cuda")
    cache = Int4KVCache.allocate(4, 16, 2, 64)
    k, v = (torch.randn(32, 2, 64, device="cuda").half() for _ in range(2))
    pages = torch.tensor([[2, 1]], **dev)
    cache.append(k, v, KVBatch(pages, torch.tensor([32], **dev), torch.tensor([0, 32], **dev), max_tokens=32))
    arrays = (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)
    before = [x.clone() for x in arrays]
    k, v = (torch.randn(count, 2, 64, device="cuda").half() for _ in range(2))
    q = torch.randn(count, 4, 64, device="cuda").half()
    table = rotary_table(64, 64)
    batch = KVBatch(pages, torch.tensor([length], **dev), torch.tensor([0, count], **dev), max_tokens=count)
    got = cache.append(k, v, batch, q=q, table=table)
    assert device_error() == 3
    places = [length - count + i for i in range(count)]
    assert [i for i, p in enumerate(places) if 0 <= p < 32] == kept
    want_k = ko.rotate(f64(k).astype(np.float32), table.cpu().numpy(), [p if 0 <= p < 64 else 0 for p in places])
    want_q = ko.rotate(f64(q).astype(np.float32), table.cpu().numpy(), [p if 0 <= p < 64 else 0 for p in places])
    held = [ko.quantise(want_k, 32), ko.quantise(f64(v).astype(np.float32), 32)]
    want = [x.cpu().numpy() for x in before]
    for i in kept:
        page, row = [2, 1][places[i] // 16], places[i] % 16
        for x, (codes, scales) in enumerate(held):
            want[2 * x][page, :, row], want[2 * x + 1][page, :, row] = ko.pack(codes[i]), scales[i]
    for x, y in zip(arrays, want):
        assert np.array_equal(x.cpu().numpy(), y)
    for i, p in enumerate(places):
        if 0 <= p < 64:  # queries turn by the same places
            assert torch.equal(got[i].cpu(), torch.from_numpy(want_q[i]).half())
    for x, (codes, scales) in zip(cache.read(batch, count), held):
        for i in range(count):
            assert np.array_equal(f64(x[i]), ko.values(codes[i], scales[i]) if i in kept else np.zeros((2, 64)))
    assert device_error() == 3


@pytest.mark.parametrize("dim, heads, counts", [(128, 4, [2, 1, 6]), (64, 8, [9, 1, 60]), (128, 8, [40, 3, 200])])
@pytest.mark.parametrize("window, causal", [(0, True), (0, False), (13, True), (5, False)])
def test_attention_beyond_the_page_table(dim, heads, counts, window, causal):
    """Tokens past the page table are not there; the queries keep the
    positions that the length gives them."""
    case = Case([48, 20, 240], counts, 2, dim, page=16, seed=dim, junk=True)
    over = [53, 20, 241]  # rows of the table for 240 tokens; the first sequence has pages for 48
    case.batch.page_table[0, 3:] = case.batch.page_table[0, 0]
    case.batch.lengths.copy_(torch.tensor(over, dtype=torch.int32))
    table = case.batch.page_table[:, :3].contiguous()
    from openquant_b200.kv_cache import KVBatch

    q = case.queries(heads, dim, torch.float16)
    for batch, caps in ((case.batch, [240, 240, 240]), (KVBatch(table, case.batch.lengths, case.batch.starts,
                                                              max_tokens=max(counts)), [48, 48, 48])):
        out, lse = case.cache.attention(q, batch, window=window, causal=causal, return_log_sum=True)
        assert device_error() == 3
        seen, rows = [], []
        for b, (n, c, cap) in enumerate(zip(over, counts, caps)):
            for p in range(n - c, n):
                hi = min(p + 1, n, cap) if causal else min(n, cap)
                lo = max(p + 1 - window, 0) if window else 0
                seen.append((b, np.arange(lo, max(hi, lo))))
                rows.append(hi <= case.lengths[b])  # (tokens 48..52 of the first sequence hold anything)
        keep = [t for t, ok in enumerate(rows) if ok]
        check_seen(case, q[keep], out[keep], lse[keep], [seen[t] for t in keep])


BAD_PAGES = [-1, 1 << 20, (1 << 31) - 1, -(1 << 31)]


@pytest.mark.parametrize("dim, group, kv_heads, heads, lengths, counts, page, window, causal", [
    (128, 32, 2, 8, [200, 37, 16, 1], [1, 1, 1, 1], 16, 0, True),       # single tokens
    (64, 64, 2, 6, [500, 90], [5, 20], 32, 70, True),                   # a few rows, a window
    (128, 128, 1, 8, [700, 90, 300], [130, 90, 1], 16, 0, True),        # prompts: the other kernel
    (64, 32, 2, 4, [900, 200], [200, 150], 48, 0, False),
    (128, 64, 1, 2, [5003], [40], 64, 0, True),                         # prompts over shared-out tokens
    (64, 32, 1, 2, [4100], [64], 16, 3000, True),
])
def test_attention_leaves_out_pages_that_are_not_there(dim, group, kv_heads, heads, lengths, counts, page, window, causal):
    """Tokens of a page number outside the cache are as if masked: page 0 does
    not stand in for them."""
    case = Case(lengths, counts, kv_heads, dim, group, page, seed=dim + heads, junk=True)
    rng = np.random.default_rng(dim)
    gone = [set() for _ in lengths]
    table = case.table.copy()
    for b, n in enumerate(lengths):
        slots = -(-n // page)
        for i in range(slots):
            if rng.random() < 0.25 or i in (slots // 2,) or table[b, i] == 0:
                table[b, i] = BAD_PAGES[rng.integers(4)]
                gone[b].add(i)
    case.batch.page_table.copy_(torch.from_numpy(table))
    q = case.queries(heads, dim, torch.float16)
    outs = []
    for junk in (1.0, float("nan")):
        case.cache.k_scales[0] = junk
        case.cache.v_scales[0] = junk
        outs.append(case.cache.attention(q, case.batch, window=window, causal=causal, return_log_sum=True))
        assert device_error() == 3
    seen = []
    for b, (n, c) in enumerate(zip(lengths, counts)):
        there = np.array([j // page not in gone[b] for j in range(n)])
        for p in range(n - c, n):
            hi = p + 1 if causal else n
            lo = max(p + 1 - window, 0) if window else 0
            idx = np.arange(lo, max(hi, lo))
            seen.append((b, idx[there[idx]]))
    check_seen(case, q, *outs[1], seen)
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])


def test_attention_leaves_out_pages_of_long_shares():
    """Forty sequences over the same pages, each without other ones of them:
    a warp's share is more blocks than one look-up covers."""
    from openquant_b200.kv_cache import KVBatch

    case = Case([2560], [40], 16, 64, page=16, junk=True)
    rng = np.random.default_rng(5)
    table = np.repeat(case.table[:1], 40, 0)
    there = rng.random(table.shape) > 0.02
    there[3] = False
    there[4] = True
    table[~there] = -1
    dev = dict(dtype=torch.int32, device="cuda")
    batch = KVBatch(torch.from_numpy(table).cuda(), torch.full((40,), 2560, **dev))
    q = case.queries(16, 64, torch.bfloat16)
    out, lse = case.cache.attention(q, batch, return_log_sum=True)
    assert device_error() == 3
    check_seen(case, q, out, lse, [(0, np.flatnonzero(np.repeat(row, 16))) for row in there])


@pytest.mark.parametrize("dim, kv_heads, heads, lengths, counts, most", [
    (128, 2, 16, [60, 90, 33], [5, 3, 4], 4),        # the longest would go to the other kernel, which is not launched
    (128, 2, 8, [700, 1, 40], [4, 1, 1], 1),         # more blocks of rows than are joined
    (64, 1, 2, [400, 300, 9], [300, 100, 9], 100),   # prompts
    (64, 1, 4, [2000, 2100, 50], [1, 2000, 1], 64),
])
def test_attention_of_more_tokens_than_max_tokens(dim, kv_heads, heads, lengths, counts, most):
    """A sequence with more of the step's tokens than the host was told is left
    out, with an error; the others are whole."""
    from openquant_b200.kv_cache import KVBatch

    case = Case(lengths, counts, kv_heads, dim, page=16, seed=most, junk=True)
    batch = KVBatch(case.batch.page_table, case.batch.lengths, case.batch.starts, max_tokens=most)
    q = case.queries(heads, dim, torch.bfloat16)
    out = torch.full_like(q, float("nan"))
    _, lse = case.cache.attention(q, batch, out=out, return_log_sum=True)
    assert device_error() == 3
    seen = []
    for b, (n, c) in enumerate(zip(lengths, counts)):
        seen += [(b, np.arange(p + 1 if c <= most else 0)) for p in range(n - c, n)]
    check_seen(case, q, out, lse, seen)


@pytest.mark.parametrize("starts, tokens, whole", [
    ([0, 5], 4, []),                 # fewer tokens in the step's arrays than starts says
    ([2, 4], 4, []),                 # the first sequence does not begin at 0
    ([0, -1, 4], 4, []),
    ([0, 2, (1 << 31) - 1], 40, [0]),
    ([-(1 << 31), 3, 6], 6, [1]),
])
@pytest.mark.parametrize("heads", [2, 16])
def test_starts_that_are_not_in_order(starts, tokens, whole, heads):
    """Such a sequence is left out, with an error: nothing is written for it,
    its rows are 0.  Sequences apart from it are whole."""
    from openquant_b200.kv_cache import Int4KVCache, KVBatch

    dev = dict(dtype=torch.int32, device="cuda")
    n = len(starts) - 1
    cache = Int4KVCache.allocate(4 * n, 16, 1, 64)
    pages = torch.arange(4 * n, **dev).view(n, 4)
    fill = torch.randn(64 * n, 1, 64, device="cuda").half()
    cache.append(fill, fill, KVBatch(pages, torch.full((n,), 64, **dev),
                                     torch.arange(n + 1, **dev) * 64, max_tokens=64))
    assert device_error() == 0
    before = [x.clone() for x in (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)]
    lengths = torch.full((n,), 50, **dev)
    batch = KVBatch(pages, lengths, torch.tensor(starts, **dev), max_tokens=40)
    k, q = torch.randn(tokens, 1, 64, device="cuda").half(), torch.randn(tokens, heads, 64, device="cuda").half()
    cache.append(k, k, batch)
    assert device_error() == 3
    own = {b: range(starts[b], starts[b + 1]) for b in whole}
    rows = torch.zeros(4 * n, 16, dtype=torch.bool, device="cuda")
    for b, r in own.items():
        for i in range(len(r)):
            j = 50 - len(r) + i
            rows[4 * b + j // 16, j % 16] = True
    for x, y in zip((cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales), before):
        assert torch.equal(x[~rows[:, None].expand(-1, 1, -1)], y[~rows[:, None].expand(-1, 1, -1)])
    got = cache.read(batch, tokens)[0]
    assert device_error() == 3
    out = torch.full_like(q, float("nan"))
    cache.attention(q, batch, out=out)
    assert device_error() == 3
    for b, r in own.items():
        one = KVBatch(pages[b:b + 1].contiguous(), lengths[:1], torch.tensor([0, len(r)], **dev), max_tokens=40)
        s = slice(r.start, r.stop)
        assert torch.equal(got[s], cache.read(one, len(r))[0])
        assert (out[s] - cache.attention(q[s], one)).abs().max() <= 2 * (2.0**-11 * 5 + 2.0**-9 * 5)
    left = torch.ones(tokens, dtype=torch.bool, device="cuda")
    for r in own.values():
        left[r.start:r.stop] = False
    assert not got[left].any()
    assert not out[left].any()
    assert device_error() == 0


@pytest.mark.parametrize("starts", [[0, 3, 2, 5], [0, 5, 1, 2, 9], [0, 9, 0, 9]])
def test_starts_of_sequences_that_overlap(starts):
    """Nothing says whose a token is: an error."""
    from openquant_b200.kv_cache import Int4KVCache, KVBatch

    dev = dict(dtype=torch.int32, device="cuda")
    n, tokens = len(starts) - 1, starts[-1]
    cache = Int4KVCache.allocate(n, 64, 1, 64)
    batch = KVBatch(torch.arange(n, **dev).view(n, 1), torch.full((n,), 50, **dev), torch.tensor(starts, **dev),
                    max_tokens=40)
    k = torch.randn(tokens, 1, 64, device="cuda").half()
    for call in (lambda: cache.append(k, k, batch), lambda: cache.read(batch, tokens),
                 lambda: cache.attention(k, batch)):
        call()
        assert device_error() == 3


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("inverse", [False, True])
def test_rotary_is_recorded_by_autograd(dtype, interleaved, inverse):
    from openquant_b200.kv_cache import rotary, rotary_table

    kw = dict(interleaved=interleaved, inverse=inverse)
    table, pos = rotary_table(300, 48, scaling={"type": "parts", "factor": 4.0, "original_positions": 256}), \
        torch.arange(9, device="cuda") * 31
    wide = torch.randn(9, 5 * 64, device="cuda").to(dtype).requires_grad_()
    x = wide.unflatten(1, (5, 64))[:, 1:4]  # strided heads
    y = rotary(x, table, pos, **kw)
    assert y.requires_grad and torch.equal(y.detach(), rotary(x.detach(), table, pos, **kw))
    g = torch.randn(9, 3, 64, device="cuda").to(dtype)
    (got,) = torch.autograd.grad(y, wide, g, retain_graph=True)
    # the formula's: the transpose, a pair (a, b) of g to (a cos + b sin, b cos - a sin)
    want = ko.rotate(f64(g).astype(np.float32), table.cpu().numpy(), pos.cpu().numpy(), interleaved, not inverse)
    got = got.unflatten(1, (5, 64))
    assert torch.equal(got[:, 1:4].cpu(), torch.from_numpy(want).to(dtype))
    assert not got[:, 0].any() and not got[:, 4].any()
    # a gradient that is one number everywhere (no stride), as sum() gives
    (ones,) = torch.autograd.grad(y.sum(), wide)
    full = ko.rotate(np.ones((9, 3, 64), np.float32), table.cpu().numpy(), pos.cpu().numpy(), interleaved, not inverse)
    assert torch.equal(ones.unflatten(1, (5, 64))[:, 1:4].cpu(), torch.from_numpy(full).to(dtype))
    if dtype is torch.float32:  # differences along a direction: the rotation is linear
        d = torch.randn(9, 3, 64, device="cuda")
        diff = (rotary(x.detach() + d, table, pos, **kw).double() - rotary(x.detach() - d, table, pos, **kw).double()) / 2
        lhs, rhs = (diff * g.double()).sum(), (d.double() * got[:, 1:4].double()).sum()
        # 1728 terms of about 1, each with a few fp32 roundings of values up to ~8
        assert abs(float(lhs - rhs)) <= 1728 * 8 * 8 * 2.0**-24
    with torch.no_grad():
        assert not rotary(x, table, pos, **kw).requires_grad
    with pytest.raises(ValueError, match="out"):
        rotary(x, table, pos, out=torch.empty_like(g), **kw)
    with pytest.raises(ValueError, match="gradient"):
        rotary(x, table.clone().requires_grad_(), pos, **kw)
    assert device_error() == 0


def test_take_device_error():
    from openquant_b200.kv_cache import rotary, rotary_table, take_device_error

    assert take_device_error() == 0
    x, table = torch.randn(1, 2, 64, device="cuda"), rotary_table(10, 64)
    rotary(x, table, torch.tensor([10], device="cuda"))
    rotary(x, table, torch.tensor([9], device="cuda"))
    assert take_device_error() == 3 and take_device_error() == 0


def test_max_tokens_beyond_32_bits_is_refused():
    from openquant_b200.kv_cache import KVBatch

    dev = dict(dtype=torch.int32, device="cuda")
    args = torch.zeros(1, 1, **dev), torch.ones(1, **dev), torch.tensor([0, 5], **dev)
    assert KVBatch(*args, max_tokens=(1 << 31) - 1).max_tokens == (1 << 31) - 1
    for n in (1 << 31, (1 << 32) + 1):  # (the second would be 1 in 32 bits)
        with pytest.raises(ValueError, match="2\\^31"):
            KVBatch(*args, max_tokens=n)


@pytest.mark.parametrize("window", [(1 << 31) - 2, (1 << 31) - 1, 1 << 31, (1 << 63) - 1, (1 << 64) + 5])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_windows_without_end(window, causal):
    """As without a window, for tokens before a sequence's start too."""
    case = Case([3, 200, 90], [3, 1, 70], 2, 64, junk=True)
    case.batch.lengths[0] = 2  # its first token is at position -1
    q = case.queries(4, 64, torch.float16)
    out, lse = case.cache.attention(q, case.batch, causal=causal, return_log_sum=True)
    got = case.cache.attention(q, case.batch, window=window, causal=causal, return_log_sum=True)
    assert torch.equal(got[0], out) and torch.equal(got[1], lse)
    seen = []
    for b, (n, c) in enumerate(zip([2, 200, 90], case.counts)):
        seen += [(b, np.arange(max(p + 1, 0) if causal else n)) for p in range(n - c, n)]
    check_seen(case, q, *got, seen)
    assert device_error() == 0


@pytest.mark.parametrize("count", [1, 200])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("scale", [1e4, -1e6, 1e7, 1e8, 1e10, 1e14, -1e20])
def test_attention_scores_beyond_fp16_and_fp32_steps(count, dim, scale):
    """Scores so large that fp32 numbers lie further apart than the weights'
    range: the largest one takes all, as far as it stands out from a score's
    error (2^-16 of scale sum |q||k| each).  Nothing overflows."""
    case = Case([700], [count], 1, dim, page=16, seed=count, junk=True)
    for dtype in (torch.float16, torch.bfloat16):
        q = case.queries(2, dim, dtype)
        out, lse = (f64(x) for x in case.cache.attention(q, case.batch, scale=scale, return_log_sum=True))
        k, v = case.sequence(0, 0)[:, 0], case.sequence(0, 1)[:, 0]
        assert np.isfinite(out).all() and np.isfinite(lse).all()
        clear = 0
        for i in range(count):
            n = 700 - count + i + 1
            for h in range(2):
                s = scale * (k[:n] @ f64(q[i, h]))
                d = 2.0**-16 * abs(scale) * (np.abs(k[:n]) @ np.abs(f64(q[i, h]))).max()
                assert abs(lse[i, h] - s.max()) <= d + 2.0**-20 * abs(s.max()) + np.log(n)
                assert (np.abs(out[i, h]) <= np.abs(v[:n]).max(0) * (1 + 2.0**-7)).all()
                best, second = np.argsort(s)[-1], np.sort(s)[-2]
                if s[best] - second > 2 * d + 60:  # the others weigh less than e^-60 together with n of them
                    clear += 1
                    tol = (U[dtype] + 2.0**-11 + 2.0**-20) * np.abs(v[best]) + 2.0**-25
                    assert (np.abs(out[i, h] - v[best]) <= tol).all()
        assert clear > count // 2
    assert device_error() == 0


@pytest.mark.parametrize("count", [1, 200])
@pytest.mark.parametrize("scale", [0.0, -0.3, 3.0, 1e9])
def test_attention_of_scales(count, scale):
    """A scale of zero (the mean of what a row sees), a negative one; equal
    scores of any size."""
    case = Case([300, 31], [count, 1], 2, 64, page=16, seed=count, junk=True)
    q = case.queries(8, 64, torch.bfloat16)
    if scale > 1:  # all keys of a head alike
        codes, scales = case.arrays[0]
        codes[:], scales[:] = codes[:1, :, :1], 1
        case.cache.k_codes.copy_(torch.from_numpy(ko.pack(codes)))
        case.cache.k_scales.copy_(torch.from_numpy(scales))
    out, lse = case.cache.attention(q, case.batch, scale=scale, return_log_sum=True)
    seen = [(b, np.arange(p + 1)) for b, (n, c) in enumerate(zip(case.lengths, case.counts)) for p in range(n - c, n)]
    if scale > 1:
        mean = np.stack([case.sequence(b, 1)[i].mean(0) for b, i in seen]).repeat(4, 1)
        spread = np.stack([np.abs(case.sequence(b, 1)[i]).mean(0) for b, i in seen]).repeat(4, 1)
        assert (np.abs(f64(out) - mean) <= 2.0**-8 * np.abs(mean) + (2.0**-11 + 2.0**-14) * spread).all()
    else:
        check_seen(case, q, out, lse, seen, scale=scale)
    assert device_error() == 0


@pytest.mark.parametrize("sequences", [33, 129, 257, 300, 513, 600, 2048])
def test_batches_of_many_sequences(sequences):
    """Sums over the sequences that take more than one pass: append, read and
    attention of many short ones, empty ones and some prompts among them."""
    from openquant_b200.kv_cache import rotary_table

    rng = np.random.default_rng(sequences)
    counts = rng.integers(0, 3, sequences)
    counts[rng.integers(0, sequences, 5)] = 40  # 80 query rows: the prompt kernel
    counts[-1] = 45
    lengths = np.where(counts > 0, counts + rng.integers(0, 30, sequences), rng.integers(0, 2, sequences) * 7)
    case = Case([int(n) for n in lengths], [int(n) for n in counts], 1, 64, page=16, seed=sequences, junk=True)
    t = case.tokens
    pad = 3
    q, k, v = (torch.randn(t + pad, h, 64, device="cuda").half() for h in (2, 1, 1))
    table = rotary_table(128, 64)
    page, row, pos = places(case)
    turned = case.cache.append(k, v, case.batch, q=q, table=table)
    want = ko.rotate(f64(q[:t]).astype(np.float32), table.cpu().numpy(), pos)
    assert torch.equal(turned[:t].cpu(), torch.from_numpy(want).half())
    refs = append_reference(case, k[:t], v[:t], 32, table, pos, False)
    for (codes, scales), (new_codes, new_scales) in zip(case.arrays, refs):
        codes[page, :, row], scales[page, :, row] = new_codes, new_scales
    for x, (codes, scales) in zip(case.cache.read(case.batch, t + pad), refs):
        assert np.array_equal(f64(x[:t]), ko.values(codes, scales)) and not x[t:].any()
    out, lse = case.cache.attention(turned, case.batch, return_log_sum=True)
    case.check(turned[:t], out[:t], lse[:t])
    assert not out[t:].any() and (lse[t:] == float("-inf")).all()


@pytest.mark.parametrize("dim, heads, length, count, window, bad", [
    (128, 8, 300, 300, 0, 100), (64, 4, 700, 200, 0, 690), (128, 4, 5003, 40, 0, 4990),   # (cut over its tokens)
    (64, 2, 5003, 64, 20, 4950), (64, 2, 5003, 64, 3000, 1960), (128, 1, 300, 300, 50, 128),
])
def test_prompts_over_a_key_that_is_not_finite(dim, heads, length, count, window, bad):
    """Rows that see it are NaN, the others are whole."""
    case = Case([length], [count], 1, dim, page=32, seed=dim, junk=True)
    where = case.table[0, bad // 32], 0, bad % 32
    for codes, scales, value in ((case.cache.k_codes, case.cache.k_scales, float("nan")),
                                 (case.cache.v_codes, case.cache.v_scales, 1.0)):
        codes[where], scales[where] = 0, value
    q = case.queries(heads, dim, torch.bfloat16)
    out, lse = case.cache.attention(q, case.batch, window=window, return_log_sum=True)
    places_of = range(length - count, length)
    sees = [p >= bad and (window == 0 or bad > p - window) for p in places_of]
    assert any(sees) and not all(sees)
    assert np.array_equal(np.isnan(f64(out)), np.broadcast_to(np.array(sees)[:, None, None], out.shape))
    assert np.array_equal(np.isnan(f64(lse)), np.broadcast_to(np.array(sees)[:, None], lse.shape))
    keep = [i for i, s in enumerate(sees) if not s]
    check_seen(case, q[keep], out[keep], lse[keep],
               [(0, np.arange(max(places_of[i] + 1 - window, 0) if window else 0, places_of[i] + 1)) for i in keep])
    assert device_error() == 0


@pytest.mark.parametrize("count", [1, 200])
@pytest.mark.parametrize("sign", [-1.0, 1.0])
def test_attention_of_bf16_queries_near_their_largest(count, sign):
    """Scores of 1e32 and more of either sign, all equal: the mean of the values."""
    case = Case([300, 31], [count, 1], 1, 64, page=16, seed=count, junk=True)
    codes, scales = case.arrays[0]
    codes[:], scales[:] = 5, 1
    case.cache.k_codes.copy_(torch.from_numpy(ko.pack(codes)))
    case.cache.k_scales.copy_(torch.from_numpy(scales))
    q = torch.full((case.tokens, 4, 64), sign * 1e31, device="cuda").bfloat16()
    out, lse = case.cache.attention(q, case.batch, return_log_sum=True)
    seen = [(b, np.arange(p + 1)) for b, (n, c) in enumerate(zip(case.lengths, case.counts)) for p in range(n - c, n)]
    mean = np.stack([case.sequence(b, 1)[i].mean(0) for b, i in seen])
    spread = np.stack([np.abs(case.sequence(b, 1)[i]).mean(0) for b, i in seen])
    assert (np.abs(f64(out) - mean) <= 2.0**-8 * np.abs(mean) + (2.0**-11 + 2.0**-14) * spread).all()
    score = float(q[0, 0, 0]) * 5 * 64 * 0.125
    assert (np.abs(f64(lse) - score) <= 2.0**-20 * abs(score)).all()
    assert device_error() == 0
