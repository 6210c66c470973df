"""4-bit key/value cache: what needs no GPU -- the rotary tables, the
quantizer's format in the oracle, and the library's refusals (which come
before any CUDA call)."""
import ctypes
import math

import numpy as np
import pytest
import torch

import kv4_oracle as ko


def test_rotary_table_is_cos_and_sin_rounded_once():
    from openquant_b200.kv_cache import rotary_table

    t = rotary_table(5000, 64, base=10000.0, device="cpu").numpy()
    i = np.arange(32)
    angle = np.arange(5000)[:, None] * 10000.0 ** (-2.0 * i / 64)
    ref = np.concatenate([np.cos(angle), np.sin(angle)], 1)
    assert t.dtype == np.float32 and t.shape == (5000, 64)
    # one rounding of values <= 1, and 5000 rad * 2^-52 of the angle twice
    np.testing.assert_allclose(t, ref, rtol=0, atol=2.0**-25 + 1e-11)


def test_rotary_scalings():
    from openquant_b200.kv_cache import _frequencies

    d, base = 128, 10000.0
    plain, one = _frequencies(d, base, None)
    assert one == 1.0
    lin, _ = _frequencies(d, base, {"type": "linear", "factor": 4.0})
    np.testing.assert_allclose(lin.numpy(), plain.numpy() / 4, rtol=1e-14)
    ntk, _ = _frequencies(d, base, {"type": "ntk", "factor": 4.0})
    # the fastest pair keeps its angle, the slowest has it divided by the factor
    assert ntk[0] == 1.0 and math.isclose(float(ntk[-1]), float(plain[-1]) / 4, rel_tol=1e-12)
    turns = 4096 * plain / (2 * math.pi)
    par, size = _frequencies(d, base, {"type": "parts", "factor": 8.0, "original_positions": 4096})
    ratio = (par / plain).numpy()
    assert (np.diff(ratio) <= 1e-15).all()
    assert (ratio[turns.numpy() > 40] == 1).all() and np.allclose(ratio[turns.numpy() < 0.9], 1 / 8)
    assert math.isclose(size, 0.1 * math.log(8) + 1)
    smo, _ = _frequencies(d, base, {"type": "smooth", "factor": 8.0, "original_positions": 4096, "low": 1, "high": 4})
    keep = np.clip((turns.numpy() - 1) / 3, 0, 1)
    np.testing.assert_allclose((smo / plain).numpy(), keep + (1 - keep) / 8, rtol=1e-12)


@pytest.mark.parametrize("scaling", [{"type": "other", "factor": 2.0}, {"type": "linear", "factor": 0.0},
                                     {"type": "smooth", "factor": 2.0, "original_positions": 8, "low": 4, "high": 4}])
def test_rotary_scaling_refusals(scaling):
    from openquant_b200.kv_cache import rotary_table

    with pytest.raises(ValueError):
        rotary_table(8, 16, scaling=scaling, device="cpu")


@pytest.mark.parametrize("positions, dim, base", [(0, 8, 1e4), (4, 7, 1e4), (4, 0, 1e4), (4, 8, -1.0)])
def test_rotary_table_refusals(positions, dim, base):
    from openquant_b200.kv_cache import rotary_table

    with pytest.raises(ValueError):
        rotary_table(positions, dim, base=base, device="cpu")


def test_cached_values_are_fp16_numbers():
    rng = np.random.default_rng(0)
    x = (rng.normal(size=(4000, 64)) * 10.0 ** rng.uniform(-7, 5, (4000, 1))).astype(np.float32)
    codes, scales = ko.quantise(x, 32)
    v = ko.values(codes, scales)
    assert np.array_equal(v, v.astype(np.float16).astype(np.float64))
    assert np.array_equal(ko.unpack(ko.pack(codes)), codes)
    # nearest of the 15 values, but for what the scale was rounded by: 2^-9 of
    # it, or half of fp16's smallest step 2^-24 (up to 0, where values read 0)
    s = np.repeat(scales.astype(np.float64), 32, -1)
    inside = np.abs(x) <= 65408
    assert (np.abs(v - x) <= np.where(codes != 0, 0.5 * s, np.minimum(0.5 * s, np.abs(x)))
            + 7 * np.maximum(2.0**-8 * s * (codes != 0), 2.0**-24))[inside].all()


def test_python_refusals_without_gpu():
    from openquant_b200.kv_cache import Int4KVCache, KVBatch, rotary

    z = torch.zeros
    with pytest.raises(ValueError, match="CUDA"):
        rotary(z(2, 2, 64), z(4, 64), z(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="3-D"):
        rotary(z(2, 64), z(4, 64), z(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="CUDA"):
        KVBatch(z(2, 2, dtype=torch.int32), z(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="int32"):
        KVBatch(z(2, 2), z(2, dtype=torch.int32))
    codes, scales = z(2, 2, 16, 64, dtype=torch.uint8), z(2, 2, 16, 4, dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        Int4KVCache(codes, scales, codes, scales)
    with pytest.raises(ValueError, match="uint8"):
        Int4KVCache(codes.int(), scales, codes, scales)
    for args in ((1, 16, 1, 96), (1, 16, 1, 128, 16), (1, 16, 1, 64, 128), (1, 24, 1, 64), (0, 16, 1, 64)):
        with pytest.raises(ValueError):
            Int4KVCache.allocate(*args, device="cpu")


@pytest.fixture(scope="module")
def lib():
    from openquant_b200 import _native, build

    build.build()
    return _native.load()


def _structs(**change):
    from openquant_b200 import kv_cache as kc

    c = dict(k_codes=1 << 20, k_scales=1 << 20, v_codes=1 << 20, v_scales=1 << 20, pages=4, page_size=16, kv_heads=2,
             head_dim=128, group_size=32)
    b = dict(page_table=1 << 20, lengths=1 << 20, starts=None, sequences=2, max_pages=2, max_tokens=1)
    for k, v in change.items():
        (c if k in c else b)[k] = v
    return kc._Cache(**c), kc._Batch(**b)


@pytest.mark.parametrize("change, message", [
    (dict(head_dim=96), "head_dim"), (dict(group_size=16), "Group size"), (dict(head_dim=64, group_size=128), "Group"),
    (dict(page_size=24), "page_size"), (dict(page_size=0), "page_size"), (dict(pages=0), "positive"),
    (dict(kv_heads=0), "positive"), (dict(k_codes=None), "null"), (dict(v_scales=(1 << 20) + 8), "aligned"),
    (dict(sequences=0), "sequences"), (dict(sequences=2049), "sequences"), (dict(max_pages=0), "page"),
    (dict(lengths=None), "null"), (dict(max_tokens=0), "max_tokens"), (dict(max_tokens=2), "starts"),
    (dict(pages=1 << 31), "large"), (dict(pages=1 << 28, kv_heads=64), "large"),
])
def test_library_refuses_bad_caches_and_batches(lib, change, message):
    from openquant_b200 import _native as nat

    c, b = _structs(**change)
    p = 1 << 20
    for st in (lib.oq_kv4_attention(ctypes.byref(c), ctypes.byref(b), p, nat.OQ_F16, 4, 512, 128, p, None, 2, 1.0, 0, 0,
                                    p, 1 << 30, None),
               lib.oq_kv4_append(ctypes.byref(c), ctypes.byref(b), None, None, 0, 0, 0, 0, 0, p, 256, 128, p, 256, 128,
                                 nat.OQ_F16, 2, None, None, 0, None),
               lib.oq_kv4_read(ctypes.byref(c), ctypes.byref(b), p, p, nat.OQ_F16, 2, None)):
        assert st == nat.OQ_ERR_INVALID and message in nat.last_error()
    assert lib.oq_kv4_attention_workspace_bytes(ctypes.byref(c), ctypes.byref(b), 4, 2) == 0


@pytest.mark.parametrize("change, message", [
    (dict(dtype=0), "fp16"), (dict(q_heads=3), "multiple"), (dict(tokens=0), "token count"), (dict(q=None), "null"),
    (dict(out=(1 << 20) + 8), "aligned"), (dict(window=-1), "window"), (dict(flags=2), "flags"),
    (dict(scale=math.inf), "finite"), (dict(ws_bytes=16), "workspace"),
])
def test_library_refuses_bad_attention_calls(lib, change, message):
    from openquant_b200 import _native as nat

    c, b = _structs()
    p = 1 << 20
    a = dict(q=p, dtype=nat.OQ_F16, q_heads=4, ts=512, hs=128, out=p, log_sum=None, tokens=2, scale=1.0, window=0,
             flags=0, ws=p, ws_bytes=1 << 30)
    a.update(change)
    st = lib.oq_kv4_attention(ctypes.byref(c), ctypes.byref(b), *a.values(), None)
    assert st == nat.OQ_ERR_INVALID and message in nat.last_error()


@pytest.mark.parametrize("change, message", [
    (dict(dtype=3), "fp32"), (dict(tokens=0), "positive"), (dict(heads=0), "positive"),
    (dict(head_dim=12), "head_dim"), (dict(head_dim=264), "head_dim"), (dict(x=None), "null"),
    (dict(positions=None), "null"), (dict(dim=7), "even"), (dict(dim=130), "at most"), (dict(rows=0), "empty"),
    (dict(table=(1 << 20) + 4), "aligned"), (dict(spec_flags=4), "flags"),
])
def test_library_refuses_bad_rotary_calls(lib, change, message):
    from openquant_b200 import _native as nat, kv_cache as kc

    p = 1 << 20
    s = dict(table=p, rows=16, dim=128, spec_flags=0)
    a = dict(x=p, y=p, dtype=nat.OQ_F16, tokens=2, heads=2, head_dim=128, positions=p)
    for k, v in change.items():
        (s if k in s else a)[k] = v
    spec = kc._RotarySpec(s["table"], s["rows"], s["dim"], s["spec_flags"])
    st = lib.oq_rotary(a["x"], a["y"], a["dtype"], a["tokens"], a["heads"], a["head_dim"], 256, 128, 256, 128,
                       ctypes.byref(spec), a["positions"], 0, None)
    assert st == nat.OQ_ERR_INVALID and message in nat.last_error()
