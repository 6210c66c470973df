"""4-bit key/value cache on the GPU against the oracle.

Rotation and quantizer: bit for bit (fp32 with one rounding per operation).

Attention, per output element:
    |error| <= max(u |o|, t) + (2^-11 + 2 d) spread + 2^-31 mass
u and t: the output type's half step, relative (2^-11 fp16, 2^-8 bf16) and at
its smallest numbers (2^-25 fp16).  spread = sum p |v| is what relative errors
of the weights p are weighted with, 2^-11 the rounding of p to fp16, and d =
2^-16 size the error of a score: at most head_dim + 8 fp32 roundings of 2^-23
(the tensor cores truncate) in sums of size <= scale * sum |q||k|; the
exponential turns d into a relative error of p and of their sum.  mass = sum
|v|: a weight below fp16's normal numbers is off by up to 2^-25 where the
largest is at least 2^6.  The log-sum: d + 2^-20 (1 + |log-sum|).
"""
import ctypes

import numpy as np
import pytest
import torch

import kv4_oracle as ko

pytestmark = pytest.mark.gpu
TINY = {torch.float16: 2.0**-25, torch.bfloat16: 0.0}
U = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}


@pytest.fixture(scope="module", autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.skip("CUDA GPU required")
    from openquant_b200 import build

    build.build()


def device_error():
    from openquant_b200 import _native as nat

    code = ctypes.c_int32(-1)
    nat.check(nat.load().oq_take_device_error(ctypes.byref(code)))
    return code.value


def f64(t):
    return t.double().cpu().numpy()


class Case:
    """Sequences with `lengths` tokens cached, the last `counts` the step's own."""

    def __init__(self, lengths, counts, kv_heads, dim, group=32, page=16, seed=0, junk=False, spare=2):
        from openquant_b200.kv_cache import Int4KVCache, KVBatch

        rng = np.random.default_rng(seed)
        self.lengths, self.counts, self.page = lengths, counts, page
        slots = max(1, max(-(-n // page) for n in lengths))
        used = sum(-(-n // page) for n in lengths)
        pages = used + spare
        order = rng.permutation(pages)
        table = np.full((len(lengths), slots), -1, np.int32)  # unused entries must not be followed
        at = 0
        for b, n in enumerate(lengths):
            c = -(-n // page)
            table[b, :c] = order[at:at + c]
            at += c
        channel = np.ones(dim)
        channel[rng.integers(0, dim, 3)] = 5
        self.arrays = []
        for ch in (channel, np.ones(dim)):
            codes, scales = ko.quantise((rng.normal(size=(pages, kv_heads, page, dim)) * ch).astype(np.float32), group)
            self.arrays.append((codes, scales))
        live = np.zeros((pages, page), bool)
        for b, n in enumerate(lengths):
            for j in range(n):
                live[table[b, j // page], j % page] = True
        if junk:  # whatever was in the memory before: NaN and infinite scales, any code
            for codes, scales in self.arrays:
                dead = np.broadcast_to(~live[:, None, :, None], scales.shape)
                scales[dead] = rng.choice(np.array([np.nan, np.inf, -np.inf, 6e4], np.float16), dead.sum())
                dead = np.broadcast_to(~live[:, None, :, None], codes.shape)
                codes[dead] = rng.integers(-8, 8, dead.sum())
        self.table = table
        dev = [torch.from_numpy(x).cuda() for c, s in self.arrays for x in (ko.pack(c), s)]
        self.cache = Int4KVCache(*dev)
        starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        self.tokens = int(starts[-1])
        self.batch = KVBatch(torch.from_numpy(table).cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(),
                             torch.from_numpy(starts).cuda(), max_tokens=max(max(counts), 1))
        self.rng = rng

    def sequence(self, b, which):
        """fp64 values [n, kv_heads, dim] of sequence b's keys (0) or values (1)."""
        codes, scales = self.arrays[which]
        n = self.lengths[b]
        pg = self.table[b, :max(1, -(-n // self.page))]
        v = ko.values(codes[pg], scales[pg])  # [pages, heads, page, dim]
        return v.transpose(0, 2, 1, 3).reshape(-1, v.shape[1], v.shape[3])[:n]

    def queries(self, heads, dim, dtype, size=1.0):
        q = self.rng.normal(size=(self.tokens, heads, dim)) * size
        return torch.from_numpy(q.astype(np.float32)).cuda().to(dtype)

    def check(self, q, out, log_sum=None, **kw):
        scale = kw.pop("scale", None) or q.shape[2] ** -0.5
        at = 0
        for b, c in enumerate(self.counts):
            if c:
                ref, lse, spread, size, mass = ko.attention(f64(q[at:at + c]), self.sequence(b, 0), self.sequence(b, 1), scale,
                                                      c, **kw)
                d = 2.0**-16 * size
                got = f64(out[at:at + c])
                tol = (np.maximum(U[out.dtype] * np.abs(ref), TINY[out.dtype])
                       + (2.0**-11 + 2 * d[..., None]) * spread + 2.0**-31 * mass + 1e-30)
                assert np.isfinite(got).all()
                bad = np.abs(got - ref) / tol
                assert bad.max() <= 1, (b, bad.max(), np.unravel_index(bad.argmax(), bad.shape))
                if log_sum is not None:
                    g = f64(log_sum[at:at + c])
                    inf = np.isinf(lse)
                    assert np.array_equal(np.isinf(g) & (g < 0), inf)
                    assert (np.abs(g - lse)[~inf] <= (d + 2.0**-20 * (1 + np.abs(lse)))[~inf]).all()
            at += c
        assert device_error() == 0


# ------------------------------------------------------------- rotary --


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens, heads, dim, rot", [(1, 1, 128, 128), (3, 5, 64, 64), (37, 9, 128, 32), (5, 3, 128, 40),
                                                     (2, 33, 96, 96), (7, 4, 256, 256), (4, 2, 8, 2), (6, 17, 64, 6)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_bits(dtype, tokens, heads, dim, rot, interleaved):
    from openquant_b200.kv_cache import rotary, rotary_table

    gen = torch.Generator(device="cuda").manual_seed(tokens + dim)
    x = torch.randn(tokens, heads, dim, device="cuda", generator=gen).to(dtype)
    table = rotary_table(70000, rot)
    pos = torch.randint(0, 70000, (tokens,), device="cuda", generator=gen)
    for p in (pos, pos.int()):
        for inverse in (False, True):
            y = rotary(x, table, p, interleaved=interleaved, inverse=inverse)
            ref = ko.rotate(x.float().cpu().numpy(), table.cpu().numpy(), pos.cpu().numpy(), interleaved, inverse)
            assert torch.equal(y.cpu(), torch.from_numpy(ref).to(dtype))
    assert device_error() == 0


def test_rotary_strided_and_in_place():
    from openquant_b200.kv_cache import rotary, rotary_table

    for dtype, width in ((torch.bfloat16, 7 * 64), (torch.float16, 7 * 64 + 3)):  # 16-byte aligned rows, and not
        base = torch.randn(11, width, device="cuda").to(dtype)
        x = base[:, :7 * 64].unflatten(1, (7, 64))[:, 1:6]
        table, pos = rotary_table(50, 64), torch.arange(11, device="cuda") * 4
        want = rotary(x.contiguous(), table, pos)
        before = base.clone()
        assert torch.equal(rotary(x, table, pos), want)
        assert rotary(x, table, pos, out=x) is x and torch.equal(x, want)
        x.copy_(before[:, :7 * 64].unflatten(1, (7, 64))[:, 1:6])
        assert torch.equal(base, before)  # nothing beside x was written
    # a rotation by 20 pairs: partners come from memory, in place too
    x = torch.randn(9, 6, 128, device="cuda")
    table = rotary_table(16, 40)
    want = rotary(x, table, torch.arange(9, device="cuda"))
    assert torch.equal(rotary(x, table, torch.arange(9, device="cuda"), out=x), want)


def test_rotary_gradient():
    """inverse=True is the gradient: <R x, g> = <x, R^T g>, and differences of
    the (linear) rotation along a direction agree with it."""
    from openquant_b200.kv_cache import rotary, rotary_table

    x, d, g = (torch.randn(8, 3, 64, device="cuda") for _ in range(3))
    table, pos = rotary_table(100, 48), torch.arange(8, device="cuda") * 12
    for inter in (False, True):
        back = rotary(g, table, pos, interleaved=inter, inverse=True)
        h = 0.5
        diff = (rotary(x + h * d, table, pos, interleaved=inter).double()
                - rotary(x - h * d, table, pos, interleaved=inter).double()) / (2 * h)
        lhs, rhs = (diff * g.double()).sum(), (d.double() * back.double()).sum()
        # 1536 terms of about 1, each with a few fp32 roundings of values up to ~8
        assert abs(float(lhs - rhs)) <= 1536 * 8 * 8 * 2.0**-24


def test_rotary_position_outside_the_table():
    from openquant_b200.kv_cache import rotary, rotary_table

    x = torch.randn(4, 2, 64, device="cuda")
    table = rotary_table(10, 64)
    out = torch.zeros_like(x)
    rotary(x, table, torch.tensor([3, 10, -1, 9], device="cuda"), out=out)
    assert device_error() == 3 and device_error() == 0
    want = rotary(x[[0, 3]].contiguous(), table, torch.tensor([3, 9], device="cuda"))
    assert torch.equal(out[[0, 3]], want) and not out[1:3].any()


def test_rotary_refusals():
    from openquant_b200.kv_cache import rotary, rotary_table

    x, t, p = torch.randn(4, 2, 64, device="cuda"), rotary_table(8, 64), torch.arange(4, device="cuda")
    for bad in (dict(x=x[..., ::2]), dict(x=x.double()), dict(x=x[:, :, :60]), dict(table=t.double()), dict(table=t.cpu()),
                dict(table=rotary_table(8, 128)), dict(positions=p[:3]), dict(positions=p.float()),
                dict(positions=p.cpu()), dict(out=x[:3]), dict(out=x.half())):
        a = dict(x=x, table=t, positions=p, out=None)
        a.update(bad)
        with pytest.raises(ValueError):
            rotary(a["x"], a["table"], a["positions"], out=a["out"])


# ------------------------------------------------------------- append --


def append_reference(case, k, v, group, table, pos, inter):
    kf, vf = k.float().cpu().numpy(), v.float().cpu().numpy()
    if table is not None:
        kf = ko.rotate(kf, table.cpu().numpy(), pos, inter)
    return ko.quantise(kf, group), ko.quantise(vf, group)


def places(case):
    """(page, row, position) of the step's tokens."""
    out = []
    for b, (n, c) in enumerate(zip(case.lengths, case.counts)):
        out += [(case.table[b, j // case.page], j % case.page, j) for j in range(n - c, n)]
    return np.array(out).T


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim, group", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)])
@pytest.mark.parametrize("kv_heads, heads, rot, inter, page", [(1, 1, None, False, 16), (2, 10, 64, False, 48),
                                                               (3, 9, 64, True, 16), (8, 64, 32, False, 64),
                                                               (5, 5, 40, False, 32)])
def test_append_bits(dtype, dim, group, kv_heads, heads, rot, inter, page):
    from openquant_b200.kv_cache import rotary_table

    case = Case([1, 17, 40, 5, 100], [1, 17, 3, 0, 33], kv_heads, dim, group, page, seed=dim + heads)
    t = case.tokens
    qkv = torch.randn(t, (heads + 2 * kv_heads) * dim, device="cuda") * 3
    qkv[2] *= 1e-6  # a token whose scales are small
    qkv = qkv.to(dtype)
    q, k, v = (x.unflatten(1, (-1, dim)) for x in qkv.split([heads * dim, kv_heads * dim, kv_heads * dim], 1))
    page_of, row, pos = places(case)
    table = rotary_table(128, rot) if rot else None
    before = [x.clone() for x in (case.cache.k_codes, case.cache.k_scales, case.cache.v_codes, case.cache.v_scales)]
    got = case.cache.append(k, v, case.batch, q=q if rot else None, table=table, interleaved=inter)
    if rot:
        want = ko.rotate(q.float().cpu().numpy(), table.cpu().numpy(), pos, inter)
        assert torch.equal(got.cpu(), torch.from_numpy(want).to(dtype))
    else:
        assert got is None
    refs = append_reference(case, k, v, group, table, pos, inter)
    now = (case.cache.k_codes, case.cache.k_scales, case.cache.v_codes, case.cache.v_scales)
    for x, (codes, scales) in enumerate(refs):
        want_codes, want_scales = before[2 * x].cpu().numpy(), before[2 * x + 1].cpu().numpy()
        want_codes[page_of, :, row], want_scales[page_of, :, row] = ko.pack(codes), scales
        # the step's rows hold the new values, and every other byte what it held
        np.testing.assert_array_equal(now[2 * x].cpu().numpy(), want_codes)
        np.testing.assert_array_equal(now[2 * x + 1].cpu().numpy().view(np.uint16), want_scales.view(np.uint16))
    for out_type in (torch.float16, torch.float32, torch.bfloat16):
        kk, vv = case.cache.read(case.batch, t, dtype=out_type)
        for x, held in ((kk, refs[0]), (vv, refs[1])):
            assert torch.equal(x.cpu(), torch.from_numpy(ko.values(*held)).to(out_type))
    assert device_error() == 0


def test_append_positions_in_place_and_unaligned():
    from openquant_b200.kv_cache import rotary_table

    case = Case([9, 30], [4, 7], 2, 128)
    table = rotary_table(500, 128)
    pos = torch.randint(0, 500, (11,), device="cuda")
    wide = torch.randn(11, 2 * 128 + 6 * 128 + 1, device="cuda").half()  # odd row pitch: no 16-byte rows
    q = wide[:, 1:1 + 768].unflatten(1, (6, 128))
    k = wide[:, 1 + 512:1 + 768].unflatten(1, (2, 128)).clone()
    v = wide[:, :256].unflatten(1, (2, 128))
    want_q = ko.rotate(q.float().cpu().numpy(), table.cpu().numpy(), pos.cpu().numpy())
    refs = append_reference(case, k, v, 32, table, pos.cpu().numpy(), False)
    v = v.clone()
    got = case.cache.append(k, v, case.batch, q=q, table=table, positions=pos, q_out=q)
    assert got is q and torch.equal(q.cpu(), torch.from_numpy(want_q).half())
    kk, vv = case.cache.read(case.batch, 11)
    assert np.array_equal(f64(kk), ko.values(*refs[0])) and np.array_equal(f64(vv), ko.values(*refs[1]))
    assert device_error() == 0


def test_append_values_that_are_not_finite():
    """The token and head of a NaN or Inf is marked through its keys; its
    neighbours are not touched, and a query that does not see it is whole."""
    case = Case([20, 20], [20, 20], 4, 64)
    k = torch.randn(40, 4, 64, device="cuda").bfloat16()
    v = torch.randn(40, 4, 64, device="cuda").bfloat16()
    k[3, 1, 5], v[7, 2, 63], k[25, 0, 0] = float("nan"), float("inf"), float("-inf")
    v[30] = 3e38  # finite: saturates
    case.cache.append(k, v, case.batch)
    kk, vv = case.cache.read(case.batch, 40, dtype=torch.float32)
    bad = np.zeros((40, 4), bool)
    bad[3, 1] = bad[7, 2] = bad[25, 0] = True
    assert np.array_equal(np.isnan(kk.cpu().numpy()).all(-1), bad) and np.array_equal(np.isnan(kk.cpu().numpy()).any(-1), bad)
    assert torch.isfinite(vv).all() and not vv[3, 1].any() and not vv[7, 2].any()
    assert (vv[30] == 7 * 9344.0).all()
    out = case.cache.attention(torch.randn(40, 4, 64, device="cuda").bfloat16(), case.batch)
    nan = np.zeros((40, 4), bool)
    nan[3:20, 1] = nan[7:20, 2] = nan[25:40, 0] = True
    got = torch.isnan(out).cpu().numpy()
    assert np.array_equal(got.all(-1), nan) and np.array_equal(got.any(-1), nan)
    assert device_error() == 0


def test_append_padding_and_bad_indices():
    from openquant_b200.kv_cache import Int4KVCache, KVBatch, rotary_table

    cache = Int4KVCache.allocate(4, 16, 1, 64)
    dev = dict(dtype=torch.int32, device="cuda")
    k = torch.randn(6, 1, 64, device="cuda").half()
    # two tokens of one sequence and four of padding
    b = KVBatch(torch.tensor([[2, 0]], **dev), torch.tensor([17], **dev), torch.tensor([0, 2], **dev), max_tokens=2)
    cache.append(k, k, b)
    assert device_error() == 0
    rows = cache.k_codes.any(-1).nonzero().tolist()
    assert rows == [[0, 0, 0], [2, 0, 15]]
    kk, vv = cache.read(b, 6)
    assert kk[:2].any() and not kk[2:].any() and not vv[2:].any()
    before = cache.k_codes.clone()
    for table, length in (([[9, 0]], 17), ([[2, -1]], 17), ([[2, 0]], 33), ([[2, 0]], 1)):
        bad = KVBatch(torch.tensor(table, **dev), torch.tensor([length], **dev), torch.tensor([0, 2], **dev),
                      max_tokens=2)
        cache.k_codes.zero_()
        cache.append(k[:2], k[:2], bad)
        assert device_error() == 3
        assert cache.k_codes.any(-1).sum() <= 1 or length == 33  # the good token of the two may be written
        cache.read(bad, 2)
        assert device_error() == 3
        cache.attention(k[:2], bad)
        code = device_error()
        assert code == 3 or length == 1  # a row before position 0 sees nothing: no error
    cache.k_codes.copy_(before)
    # a rotation beyond the table
    cache.append(k[:2], k[:2], b, table=rotary_table(16, 64))
    assert device_error() == 3


# ---------------------------------------------------------- attention --


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim, group", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)])
@pytest.mark.parametrize("kv_heads, heads", [(1, 1), (2, 16), (3, 15), (1, 24)])
def test_attention_single_tokens(dtype, dim, group, kv_heads, heads):
    lengths = [1, 15, 16, 17, 63, 64, 65, 200, 129, 2]
    case = Case(lengths, [1] * len(lengths), kv_heads, dim, group, page=16, seed=dim + heads, junk=True)
    q = case.queries(heads, dim, dtype)
    out, lse = case.cache.attention(q, case.batch, return_log_sum=True)
    case.check(q, out, lse)


def test_attention_batch_without_starts_and_outputs():
    from openquant_b200.kv_cache import KVBatch

    case = Case([33, 100, 7], [1, 1, 1], 2, 128, page=32, junk=True)
    batch = KVBatch(case.batch.page_table, case.batch.lengths)
    q = case.queries(4, 128, torch.bfloat16)
    out = torch.full_like(q, float("nan"))
    assert case.cache.attention(q, batch, out=out) is out
    case.check(q, out)
    # a strided view of a fused projection gives the same bits, aligned or not
    for extra in (0, 3):
        wide = torch.randn(3, 4 * 128 + 2 * 128 + extra, device="cuda").bfloat16()
        view = wide[:, extra:extra + 512].unflatten(1, (4, 128))
        view.copy_(q)
        assert torch.equal(case.cache.attention(view, batch), out)


@pytest.mark.parametrize("page", [16, 48, 128])
@pytest.mark.parametrize("window, causal", [(0, True), (0, False), (1, True), (20, True), (100, True), (70, False)])
def test_attention_masks(page, window, causal):
    case = Case([90, 5, 300, 64, 1, 161], [7, 5, 2, 1, 1, 40], 2, 64, page=page, seed=window, junk=True)
    q = case.queries(6, 64, torch.float16, size=2.0)
    out, lse = case.cache.attention(q, case.batch, window=window, causal=causal, return_log_sum=True)
    case.check(q, out, lse, window=window, causal=causal)


def test_attention_window_with_freed_pages():
    """Pages below every window may be gone: their entries are not followed."""
    case = Case([400, 320], [3, 1], 2, 128, page=16, junk=True)
    q = case.queries(4, 128, torch.float16)
    for b, (n, c) in enumerate(zip(case.lengths, case.counts)):
        gone = (n - c + 1 - 50) // 16
        case.batch.page_table[b, :gone] = -1
    out = case.cache.attention(q, case.batch, window=50)
    case.check(q, out, window=50)


def test_attention_rows_that_see_nothing():
    """Lengths of zero and tokens before a sequence's start (more tokens than
    its length): 0 and -inf, beside rows that see something; padding too."""
    from openquant_b200.kv_cache import KVBatch

    case = Case([0, 3, 40], [2, 3, 1], 2, 64, junk=True)
    dev = dict(dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 2, 7, 8], **dev)  # the second has 5 tokens for a length of 3
    batch = KVBatch(case.batch.page_table, case.batch.lengths, starts, max_tokens=5)
    q = torch.randn(11, 4, 64, device="cuda").half()
    out, lse = case.cache.attention(q, batch, return_log_sum=True)
    empty = [0, 1, 2, 3, 8, 9, 10]
    assert not out[empty].any() and (lse[empty] == float("-inf")).all()
    case.counts = [0, 3, 1]
    case.check(q[[4, 5, 6, 7]], out[[4, 5, 6, 7]], lse[[4, 5, 6, 7]])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kv_heads, heads, dim, lengths, counts", [
    (2, 2, 128, [300], [300]),              # a whole prompt
    (1, 8, 128, [700], [130]),              # a chunk over what is cached
    (2, 14, 64, [150, 1, 260, 90], [150, 1, 33, 2]),   # mixed: prompt, step, chunk, drafts
    (4, 4, 64, [513, 257], [257, 129]),
    (1, 5, 128, [1000, 31], [60, 31]),
])
def test_attention_chunks(dtype, kv_heads, heads, dim, lengths, counts):
    case = Case(lengths, counts, kv_heads, dim, group=64, page=32, seed=heads, junk=True)
    q = case.queries(heads, dim, dtype)
    out, lse = case.cache.attention(q, case.batch, return_log_sum=True)
    case.check(q, out, lse)
    out = case.cache.attention(q, case.batch, window=77, scale=0.2)
    case.check(q, out, window=77, scale=0.2)


def test_attention_long_context():
    case = Case([20011, 3], [1, 1], 1, 128, group=128, page=64, junk=True)
    q = case.queries(8, 128, torch.bfloat16)
    out, lse = case.cache.attention(q, case.batch, return_log_sum=True)
    case.check(q, out, lse)


@pytest.mark.parametrize("lengths, counts, window", [([5003], [40], 0), ([4100, 700, 130], [33, 64, 129], 0),
                                                     ([3000, 2999], [300, 1], 1500)])
def test_attention_few_rows_over_long_contexts(lengths, counts, window):
    """Too few rows for the GPU: their cached tokens are shared out and joined."""
    case = Case(lengths, counts, 1, 64, page=32, junk=True)
    q = case.queries(2, 64, torch.float16)
    out, lse = case.cache.attention(q, case.batch, window=window, return_log_sum=True)
    case.check(q, out, lse, window=window)


@pytest.mark.parametrize("count", [1, 200])
def test_attention_scores_far_apart(count):
    """Scores that grow along the sequence (the running maximum is raised again
    and again), and very large and very small queries."""
    case = Case([400], [count], 1, 64, page=16)
    codes, scales = case.arrays[0]
    for j in range(400):
        scales[case.table[0, j // 16], 0, j % 16] = ko.bf16((j + 1) / 32)  # 8 significant bits, as the format has
    case.cache.k_scales.copy_(torch.from_numpy(scales))
    for size, dtype in ((3.0, torch.float16), (1e-3, torch.float16), (300.0, torch.bfloat16), (1e-30, torch.bfloat16)):
        q = case.queries(3, 64, dtype, size=size)
        scale = 0.125 if size < 100 else 0.125 / 100
        out, lse = case.cache.attention(q, case.batch, scale=scale, return_log_sum=True)
        case.check(q, out, lse, scale=scale)


def test_attention_offsets_beyond_32_bits():
    """A cache of more than 2^31 code bytes, its last pages in use."""
    from openquant_b200.kv_cache import Int4KVCache, KVBatch

    pages, page, heads, dim = 33000, 64, 16, 128
    assert pages * page * heads * dim // 2 > 1 << 31
    cache = Int4KVCache.allocate(pages, page, heads, dim, 128)
    small = Int4KVCache.allocate(4, page, heads, dim, 128)
    dev = dict(dtype=torch.int32, device="cuda")
    far = KVBatch(torch.tensor([[pages - 1, 5, pages - 2]], **dev), torch.tensor([150], **dev),
                  torch.tensor([0, 150], **dev), max_tokens=150)
    near = KVBatch(torch.tensor([[3, 0, 1]], **dev), torch.tensor([150], **dev), torch.tensor([0, 150], **dev),
                   max_tokens=150)
    k, v = (torch.randn(150, heads, dim, device="cuda").half() for _ in range(2))
    q = torch.randn(150, heads, dim, device="cuda").half()
    for c, b in ((cache, far), (small, near)):
        c.append(k, v, b)
    for x, y in zip(cache.read(far, 150), small.read(near, 150)):
        assert torch.equal(x, y)
    assert torch.equal(cache.attention(q, far), small.attention(q, near))
    assert device_error() == 0


def test_attention_is_deterministic_on_streams_and_in_graphs():
    case = Case([700, 80, 33], [1, 3, 33], 2, 128, junk=True)
    q = case.queries(8, 128, torch.float16)
    first = case.cache.attention(q, case.batch)
    case.check(q, first)
    assert all(torch.equal(first, case.cache.attention(q, case.batch)) for _ in range(5))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = case.cache.attention(q, case.batch)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, first)
    graph = torch.cuda.CUDAGraph()
    out = torch.empty_like(q)
    with torch.cuda.graph(graph):
        case.cache.attention(q, case.batch, out=out)
    # the graph reads the lengths when it runs
    case.batch.lengths.copy_(torch.tensor([500, 80, 33], dtype=torch.int32))
    graph.replay()
    case.lengths = [500, 80, 33]
    case.check(q, out)


def test_decode_loop_matches_attention_on_the_whole():
    """Tokens appended one by one and attended as they come give the rows of
    the same prompt in one chunk."""
    from openquant_b200.kv_cache import Int4KVCache, KVBatch, rotary_table

    dev = dict(dtype=torch.int32, device="cuda")
    table = rotary_table(64, 64)
    q, k, v = (torch.randn(40, h, 64, device="cuda").half() for h in (6, 2, 2))
    pages = torch.tensor([[3, 1, 0]], **dev)
    one, whole = (Int4KVCache.allocate(4, 16, 2, 64) for _ in range(2))
    chunk = KVBatch(pages, torch.tensor([40], **dev), torch.tensor([0, 40], **dev), max_tokens=40)
    ref = whole.attention(whole.append(k, v, chunk, q=q, table=table), chunk)
    for j in range(40):
        step = KVBatch(pages, torch.tensor([j + 1], **dev))
        s = slice(j, j + 1)
        y = one.attention(one.append(k[s], v[s], step, q=q[s], table=table), step)
        # two orders of the same sums: twice the bound of one, with spread <= max |v| ~ 4
        assert (y - ref[s]).abs().max() <= 2 * (2.0**-11 * 4 + 2.0**-9 * 4)
    for x, y in zip((one.k_codes, one.k_scales, one.v_codes, one.v_scales),
                    (whole.k_codes, whole.k_scales, whole.v_codes, whole.v_scales)):
        assert torch.equal(x, y)


def test_refusals():
    from openquant_b200.kv_cache import Int4KVCache, KVBatch, rotary_table

    dev = dict(dtype=torch.int32, device="cuda")
    cache = Int4KVCache.allocate(4, 16, 2, 64)
    t, n = torch.zeros(2, 2, **dev), torch.ones(2, **dev)
    batch = KVBatch(t, n)
    k, q = torch.randn(2, 2, 64, device="cuda").half(), torch.randn(2, 4, 64, device="cuda").half()
    table = rotary_table(16, 64)
    for bad in (lambda: KVBatch(t, n[:1]), lambda: KVBatch(t, n, torch.zeros(2, **dev), max_tokens=1),
                lambda: KVBatch(t, n, torch.zeros(3, **dev)), lambda: KVBatch(t.T, n), lambda: KVBatch(t, n.long()),
                lambda: KVBatch(t, n, max_tokens=2), lambda: KVBatch(t.cpu(), n),
                lambda: KVBatch(torch.zeros(2049, 1, **dev), torch.zeros(2049, **dev)),
                lambda: Int4KVCache(cache.k_codes, cache.k_scales[:, :1], cache.v_codes, cache.v_scales[:, :1]),
                lambda: Int4KVCache(cache.k_codes[:, :, ::2], cache.k_scales, cache.v_codes, cache.v_scales),
                lambda: cache.append(k[:, :1], k[:, :1], batch), lambda: cache.append(k.float(), k.float(), batch),
                lambda: cache.append(k, k[:1], batch), lambda: cache.append(k, k.bfloat16(), batch),
                lambda: cache.append(k, k, batch, q=q), lambda: cache.append(k, k, batch, q=q[:1], table=table),
                lambda: cache.append(k, k, batch, q=q.bfloat16(), table=table),
                lambda: cache.append(k, k, batch, q_out=q), lambda: cache.append(k, k, batch, table=rotary_table(4, 128)),
                lambda: cache.append(k, k, batch, table=table, positions=torch.zeros(3, **dev)),
                lambda: cache.append(k.transpose(0, 2), k.transpose(0, 2), batch), lambda: cache.append(k, k, t),
                lambda: cache.read(batch, 0), lambda: cache.read(batch, 2, dtype=torch.int8),
                lambda: cache.attention(q[..., :32], batch), lambda: cache.attention(q[:, :3], batch),
                lambda: cache.attention(q.float(), batch), lambda: cache.attention(q, batch, window=-1),
                lambda: cache.attention(q, batch, scale=float("nan")), lambda: cache.attention(q, batch, out=q[:1]),
                lambda: cache.attention(q, batch, out=q.transpose(0, 1)), lambda: cache.attention(q.cpu(), batch)):
        with pytest.raises(ValueError):
            bad()
    torch.cuda.synchronize()
    assert device_error() == 0


def test_example_layer_decodes_over_what_it_cached():
    """examples/kv_cache_decode.py: the last captured step's attention against
    the oracle on the values that the cache holds."""
    import os
    import sys

    from conftest import ROOT
    from openquant_b200.kv_cache import KVBatch

    sys.path.insert(0, os.path.join(ROOT, "examples"))
    import kv_cache_decode as ex

    layer, batch, _ = ex.run(requests=3, prompt=50, steps=5, heads=6, kv_heads=2, head_dim=64, page_size=16)
    q, y = layer.last
    lengths = batch.lengths.tolist()
    starts = torch.tensor([0, *np.cumsum(lengths)], dtype=torch.int32).cuda()
    whole = KVBatch(batch.page_table, batch.lengths, starts, max_tokens=max(lengths))
    k, v = (f64(x) for x in layer.cache.read(whole, sum(lengths)))
    for b, n in enumerate(lengths):
        s = slice(int(starts[b]), int(starts[b + 1]))
        ref, _, spread, size, mass = ko.attention(f64(q[b:b + 1]), k[s], v[s], 64**-0.5, 1)
        tol = (np.maximum(2.0**-11 * np.abs(ref), TINY[torch.float16]) + (2.0**-11 + 2.0**-15 * size[..., None]) * spread
               + 2.0**-31 * mass)
        assert (np.abs(f64(y[b:b + 1]) - ref) <= tol).all()
    assert device_error() == 0
