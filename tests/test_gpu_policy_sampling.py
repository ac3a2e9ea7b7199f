"""GPU parity of policy sampling against the float64 oracle (oracle/policy.py).

Token ids, accepted lengths and status words are whole numbers and must be equal, but for one
case. The kernel's float64 sums are trees, the oracle's sequential; each is within (n - 1) 2^-53
of the exact sum of n weights, relative (every addition rounds by at most 2^-53 and no weight is
negative). So where u times the total lies within 2 n 2^-53 of the total from the boundary
between two kept ids, either of the two is right: rows made of a few repeated values reach that
(four ids of weight 1, 2812 of weight e^-2 and u = 1/4 put it on the boundary exactly). The
weights max(p - q, 0) of a refused draft have errors of their own, at most 4 2^-53 p each (the
weight, the total, the quotient, the difference), so there the bound is 2 (n + 4) 2^-53 of p's
whole mass, which is 1.

Probabilities are float64 values rounded once to float32: within 2^-24 of the oracle's,
relative, plus its sums' error and, below float32's smallest normal number, 2^-150."""

from __future__ import annotations

import ctypes
import decimal
import math

import numpy as np
import pytest
import torch

import onyx_b200 as ox
from onyx_b200 import _lib, workloads
from oracle import policy as opol
from oracle import sampling as osamp
from tests.gpu_util import host, masks_to_device, requires_cuda, to_device

pytestmark = [pytest.mark.gpu, requires_cuda]

POLICIES = {
    "plain": (1.0, 0, 1.0, 0.0),
    "greedy": (0.0, 7, 0.5, 0.3),
    "top_k": (0.9, 50, 1.0, 0.0),
    "top_k1": (1.0, 1, 1.0, 0.0),
    "top_p": (0.8, 0, 0.9, 0.0),
    "top_p_small": (1.0, 0, 0.02, 0.0),
    "top_p_hot": (2.0, 0, 0.99, 0.0),
    "min_p": (1.0, 0, 1.0, 0.05),
    "min_p_all": (1.0, 0, 1.0, 1.0),
    "all": (0.7, 40, 0.95, 0.02),
    "k_wide": (1.5, 1000, 0.9, 0.0),
}


def f64(x: np.ndarray, dtype: str) -> np.ndarray:
    if dtype == "bf16":
        return (x.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return x.astype(np.float64)


def rounded(x: np.ndarray, dtype: str) -> np.ndarray:
    x = np.asarray(x, np.float32)
    return workloads.bf16_bits(x) if dtype == "bf16" else x.astype(
        np.float16 if dtype == "f16" else np.float32)


def normal(rng, shape, dtype, scale=3.0):
    return rounded(rng.standard_normal(shape) * scale, dtype)


def table(policy, rows):
    return np.tile(np.asarray(policy, np.float64), (rows, 1))


def gpu(a, dtype=torch.float64):
    return torch.as_tensor(np.asarray(a), dtype=dtype).cuda()


def assert_probs(got: torch.Tensor, expected: np.ndarray):
    got = host(got).astype(np.float64)
    np.testing.assert_array_equal(got > 0, expected.astype(np.float32) > 0)
    err = np.abs(got - expected)
    assert (err <= expected * (2.0**-24 + 1e-10) + 2.0**-150).all(), err.max()


def on_boundary(w, u, a: int, b: int) -> bool:
    """Whether rounding decides between the ids a and b of the weights w (the module's bound;
    weights max(p - q, 0) sum to less than 1, all others to at least 1)."""
    ids = np.flatnonzero(w)
    at = np.searchsorted(ids, min(a, b))
    if at + 1 >= ids.size or (ids[at], ids[at + 1]) != (min(a, b), max(a, b)):
        return False
    cum = np.cumsum(w[ids])
    return abs(cum[at] - u * cum[-1]) <= 2 * (ids.size + 4) * 2.0**-53 * max(1.0, cum[-1])


def check(x, m, dtype, policies, u, *, probs=True):
    """Draw and probabilities of oracle-layout rows against the oracle."""
    xt, mt = to_device(x, dtype), None if m is None else masks_to_device(m)
    pol = gpu(policies)
    r = ox.policy_sample(xt, mt, pol, torch.as_tensor(u).cuda())
    v = f64(x, dtype)
    ids, status = opol.sample(v, m, policies, np.asarray(u, np.float64))
    np.testing.assert_array_equal(host(r.status).astype(np.uint32), status)
    got = host(r.token_ids)
    for i in np.flatnonzero(got != ids):
        valid = np.ones(v.shape[1], bool) if m is None else osamp.unpack_mask(m[i], v.shape[1])
        w = opol.kept_weights(v[i], valid, policies[i])[1]
        assert on_boundary(w, float(u[i]), got[i], ids[i]), (i, got, ids)
    if probs:
        p, st = ox.policy_probs(xt, mt, pol)
        p_ref, st_ref = opol.probs(v, m, policies)
        np.testing.assert_array_equal(host(st).astype(np.uint32), st_ref)
        assert_probs(p, p_ref)
    return host(r.token_ids)


@pytest.mark.parametrize("policy", list(POLICIES))
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_random_rows(dtype, policy, cuda_lib):
    rng = np.random.default_rng(len(dtype) * 100 + list(POLICIES).index(policy))
    rows, vocab = 12, 5003
    x = normal(rng, (rows, vocab), dtype)
    m = workloads.bernoulli_masks(rng, rng.uniform(0.002, 0.5, rows), vocab)
    check(x, m, dtype, table(POLICIES[policy], rows), rng.random(rows))
    check(x, None, dtype, table(POLICIES[policy], rows), rng.random(rows, dtype=np.float32))


@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 9, 31, 33, 255, 256, 257, 4095, 4097, 8193, 32769])
def test_odd_vocabularies(vocab, cuda_lib):
    """Rows that end inside a vector, a mask word, a chunk and a CTA's part."""
    rng = np.random.default_rng(vocab)
    for dtype, rows in (("bf16", 3), ("f32", 1)):
        x = normal(rng, (rows, vocab), dtype)
        m = workloads.bernoulli_masks(rng, np.full(rows, 0.7), vocab)
        for policy in ("plain", "all", "top_p", "greedy"):
            check(x, m, dtype, table(POLICIES[policy], rows), rng.random(rows))
            check(x, None, dtype, table(POLICIES[policy], rows), rng.random(rows))


@pytest.mark.parametrize("rows", [1, 2, 5, 16, 40, 75, 149, 300])
def test_batches(rows, cuda_lib):
    """Every cluster size, each row under a policy of its own."""
    rng = np.random.default_rng(rows)
    vocab = 40000 if rows <= 40 else 9001
    x = normal(rng, (rows, vocab), "bf16")
    m = workloads.bernoulli_masks(rng, rng.uniform(0.01, 0.9, rows), vocab)
    names = list(POLICIES)
    policies = np.stack([POLICIES[names[i]] for i in rng.integers(0, len(names), rows)])
    check(x, m, "bf16", policies, rng.random(rows))


def test_full_vocabulary_rows(cuda_lib):
    w = workloads.batched(rows=6)
    rng = np.random.default_rng(6)
    for policy in ("top_p", "all", "plain", "top_p_hot", "k_wide"):
        check(w["logits_bf16"], w["masks"], "bf16", table(POLICIES[policy], 6), rng.random(6))
        check(w["logits_bf16"][:3], None, "bf16", table(POLICIES[policy], 3), rng.random(3))


def test_rows_longer_than_shared_memory(cuda_lib):
    rng = np.random.default_rng(8)
    for dtype in ("f32", "bf16"):
        x = normal(rng, (2, 1500001), dtype)
        check(x, None, dtype, np.stack([POLICIES["top_p"], POLICIES["all"]]), rng.random(2))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_wide_value_ranges(dtype, cuda_lib):
    """Values from a hundredth to thousands, temperatures from 0.001 to 1000."""
    rng = np.random.default_rng(77)
    scales = np.array([[0.01], [0.3], [1.0], [8.0], [30.0], [3000.0], [1e-6], [3.0]])
    x = rounded(rng.standard_normal((8, 9001)) * scales, dtype)
    m = workloads.bernoulli_masks(rng, rng.uniform(0.05, 1.0, 8), 9001)
    for policy in ((1000.0, 0, 0.9, 0.0), (5.0, 0, 0.999, 0.0), (0.001, 0, 0.5, 0.0),
                   (0.05, 200, 0.95, 0.0), (1000.0, 3000, 0.7, 0.0), (1.0, 0, 0.5, 1e-6),
                   (1e-310, 0, 0.9, 0.0), (50.0, 5, 1.0, 0.99)):
        check(x, m, dtype, table(policy, 8), rng.random(8))
        check(x, None, dtype, table(policy, 8), rng.random(8))


def test_extreme_finite_values(cuda_lib):
    """The largest and lowest finite values of a type, as masks of other programs write them."""
    for dtype, big in (("f32", 3.4028234e38), ("f16", 65504.0), ("bf16", 3.3895314e38)):
        x = np.zeros((3, 700), np.float32)
        x[:, 100:] = -big
        x[0, :100] = np.linspace(-3, 3, 100)
        x[1, :] = -big  # nothing but the lowest value: a flat row
        x[2, 5] = big
        x = rounded(x, dtype)
        for policy in ("plain", "top_p", "all", "top_k"):
            check(x, None, dtype, table(POLICIES[policy], 3), [0.1, 0.5, 0.9])


def test_special_rows(cuda_lib):
    vocab = 300
    rng = np.random.default_rng(3)
    x = (rng.standard_normal((12, vocab)) * 2).astype(np.float32)
    m = np.full((12, (vocab + 31) // 32), 0xFFFFFFFF, np.uint32)
    x[0, [3, 40, 41, 299]] = 50.0            # ties among the leaders
    x[1, [7, 100, 101, 280]] = np.inf        # +inf ids share the mass
    x[2, 17] = np.nan                        # a valid NaN
    x[3, :] = -np.inf
    m[4, :] = 0                              # no valid id
    m[4, -1] = np.uint32(0xFFFFFFFF) << np.uint32(vocab % 32)  # bits past the vocabulary only
    x[5, :] = 0.5                            # flat
    x[6, ::3] = -np.inf
    x[7, 250] = 1e30                         # one id takes all the mass
    x[8, [0, 31, 299]] = [np.nan, np.inf, -np.inf]
    m[8] = 0
    m[8, 0] = 0b110                          # NaN and infinities in masked places
    x[9, :] = -0.0
    x[9, ::2] = 0.0                          # signed zeros tie
    m[10] = 0
    m[10, 9] = 1 << 11                       # the last id alone
    x[11, [20, 200]] = [np.inf, np.nan]
    for policy in list(POLICIES.values()) + [(1.0, 2, 1.0, 0.0), (1.0, 3, 0.5, 0.0)]:
        for u in (0.0, 0.3, 0.74, 1.0 - 2.0**-24):
            check(x, m, "f32", table(policy, 12), np.full(12, u, np.float32))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_ties_at_the_cut(dtype, cuda_lib):
    """Thousands of ids share the value the cut falls on: the first in id order are kept."""
    vocab = 20000
    x = np.full((4, vocab), -5.0, np.float32)
    x[:, ::7] = 1.0
    x[1, 100] = 2.0
    x[2, ::5000] = 3.0
    x[3, :] = 0.25
    x = rounded(x, dtype)
    for policy in ((1.0, 0, 0.1, 0.0), (1.0, 0, 0.5, 0.0), (1.0, 0, 0.97, 0.0), (1.0, 5, 1.0, 0.0),
                   (1.0, 1000, 1.0, 0.0), (1.0, 2861, 0.9, 0.0), (1.0, 19999, 0.5, 0.2)):
        for u in (0.0, 0.25, 0.6, 0.999):
            check(x, None, dtype, table(policy, 4), np.full(4, u), probs=u == 0.25)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_ways_to_the_cut(dtype, cuda_lib):
    """Rows and policies that take each way to the cut: log-probabilities (all negative), one id
    far above the rest, most ids at the type's lowest value, values next to zero, steps of many
    equal values, wide and narrow ones; temperatures that keep one id and tens of thousands;
    top-k below, at and past the lengths of the lists."""
    rng = np.random.default_rng(70 + len(dtype))
    vocab = 30011
    x = rng.standard_normal((9, vocab)) * 3
    x[1] -= np.log(np.exp(x[1]).sum()) + 30
    x[2, 12345] = 45.0
    x[3, rng.random(vocab) < 0.8] = -65504.0
    x[4] *= 1e-4
    x[5] = np.round(x[5])
    x[6] *= 20
    x[7] = rng.random(vocab) * 0.1 + 200.0
    x[8, :20000] = -np.inf
    x = rounded(x, dtype)
    m = workloads.bernoulli_masks(rng, np.full(9, 0.3), vocab)
    for policy in ((0.8, 0, 0.9, 0.0), (1.2, 0, 0.95, 0.0), (3.0, 0, 0.99, 0.0), (0.05, 0, 0.9, 0.0),
                   (1.0, 512, 0.9, 0.0), (1.0, 513, 0.9, 0.0), (1.0, 1500, 1.0, 0.0),
                   (2.0, 5000, 0.7, 0.01), (1.0, 0, 0.999999, 0.0), (0.7, 3, 0.5, 0.0)):
        check(x, None, dtype, table(policy, 9), rng.random(9), probs=policy[0] != 3.0)
        check(x, m, dtype, table(policy, 9), rng.random(9), probs=policy[0] == 2.0)


def test_rows_past_the_peaks(cuda_lib):
    """2.2 million ids: parts of a row too long for their peaks, read whole in every pass."""
    rng = np.random.default_rng(81)
    for dtype in ("bf16", "f32"):
        x = normal(rng, (1, 2_200_003), dtype)
        check(x, None, dtype, table(POLICIES["top_p"], 1), rng.random(1), probs=False)
        check(x, None, dtype, table(POLICIES["all"], 1), rng.random(1), probs=False)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_rows_of_every_alignment(dtype, cuda_lib):
    """Rows that follow each other without padding start at every offset from 16 bytes."""
    rng = np.random.default_rng(90)
    for vocab in (1001, 20003, 70001):
        x = normal(rng, (9, vocab), dtype)
        m = workloads.bernoulli_masks(rng, rng.uniform(0.1, 0.9, 9), vocab)
        for policy in ("top_p", "all", "plain"):
            check(x, m, dtype, table(POLICIES[policy], 9), rng.random(9), probs=policy == "all")
            check(x, None, dtype, table(POLICIES[policy], 9), rng.random(9), probs=False)


def test_nearly_equal_float32_values(cuda_lib):
    """float32 values that agree in all but their last bits, thousands in the same place."""
    rng = np.random.default_rng(12)
    x = np.full((3, 30000), 7.0, np.float32)
    x += rng.integers(0, 64, x.shape).astype(np.float32) * np.float32(2.0**-21)
    x[1] = -x[1]
    x[2] = x[2] * np.float32(2.0**-20)
    for policy in ((1.0, 0, 0.5, 0.0), (1.0, 12345, 0.9, 0.0), (1e-6, 0, 0.3, 0.0),
                   (1.0, 100, 1.0, 0.0)):
        check(x, None, "f32", table(policy, 3), rng.random(3))


def test_edge_numbers(cuda_lib):
    """u = 0 draws the first kept id, u next to 1 the last that rounding allows."""
    rng = np.random.default_rng(9)
    x = normal(rng, (6, 2000), "bf16")
    for dtype in (np.float32, np.float64):
        for u in (0.0, np.nextafter(dtype(1), dtype(0)), np.finfo(dtype).tiny):
            check(x, None, "bf16", table(POLICIES["top_p"], 6), np.full(6, u, dtype))


def test_bad_policies_and_numbers_are_reported(cuda_lib):
    rng = np.random.default_rng(10)
    bad = [(-1, 0, 1, 0), (np.nan, 0, 1, 0), (np.inf, 0, 1, 0), (1, -1, 1, 0), (1, 1.5, 1, 0),
           (1, np.nan, 1, 0), (1, 0, 0, 0), (1, 0, 1.1, 0), (1, 0, np.nan, 0), (1, 0, 1, -0.1),
           (1, 0, 1, 1.1), (1, 0, 1, np.nan), (1, np.inf, 1, 0), (1, 1e300, 1, 0), (1, 0, 1, 0)]
    n = len(bad)
    x = normal(rng, (n, 900), "f32")
    x[0] = np.nan  # not looked at
    check(x, None, "f32", np.asarray(bad, np.float64), np.full(n, 0.5))
    u = np.array([1.0, -0.1, np.nan, np.inf, 0.5] * 3)
    check(x[1:], None, "f32", table(POLICIES["plain"], n - 1), u[: n - 1], probs=False)
    r = ox.policy_sample(to_device(x[1:3], "f32"), None, gpu(table(POLICIES["plain"], 2)),
                         gpu([1.0, 0.5]))
    assert host(r.status).tolist() == [ox.STATUS_BAD_POLICY, 0]


def test_strides(cuda_lib):
    """Column slices, padded and repeated rows, wide policy tables, strided numbers."""
    rng = np.random.default_rng(5)
    full = normal(rng, (4, 3011), "bf16")
    m = workloads.bernoulli_masks(rng, np.array([0.5, 0.1, 1.0, 0.02]), 3000)
    policies = np.stack([POLICIES[n] for n in ("top_p", "all", "plain", "top_k")])
    u = rng.random(4)
    wide = torch.zeros(4, 6, dtype=torch.float64, device="cuda")
    wide[:, :4] = gpu(policies)
    us = torch.zeros(4, 3, dtype=torch.float64, device="cuda")
    us[:, 1] = gpu(u)
    for off in (0, 1, 3, 8, 11):
        x = np.ascontiguousarray(full[:, off:off + 3000])
        r = ox.policy_sample(to_device(full, "bf16")[:, off:off + 3000], masks_to_device(m),
                             wide[:, :4], us[:, 1])
        ids, status = opol.sample(f64(x, "bf16"), m, policies, u)
        np.testing.assert_array_equal(host(r.token_ids), ids)
        np.testing.assert_array_equal(host(r.status).astype(np.uint32), status)
        out = torch.full((4, 3009), 7.0, device="cuda")
        p, _ = ox.policy_probs(to_device(full, "bf16")[:, off:off + 3000], masks_to_device(m),
                               wide[:, :4], out=out[:, 4:3004])
        assert p.data_ptr() == out[:, 4:].data_ptr()
        assert_probs(p, opol.probs(f64(x, "bf16"), m, policies)[0])
        assert (host(out[:, :4]) == 7).all() and (host(out[:, 3004:]) == 7).all()
    # one row seen four times, one mask row, one policy, one number; transposed logits
    row = to_device(full[:1, :3000], "bf16")
    one = ox.policy_sample(row.expand(4, 3000), masks_to_device(m[:1]).expand(4, -1),
                           gpu(policies[0]), gpu(u[:1]).expand(4))
    ref = opol.sample(f64(full[:1, :3000], "bf16"), m[:1], policies[:1], u[:1])[0]
    assert host(one.token_ids).tolist() == [int(ref[0])] * 4
    t = to_device(full[:, :3000], "bf16").t().contiguous().t()
    r = ox.policy_sample(t, masks_to_device(m), gpu(policies), gpu(u))
    np.testing.assert_array_equal(
        host(r.token_ids), opol.sample(f64(full[:, :3000], "bf16"), m, policies, u)[0])
    # a single row [V]
    r = ox.policy_sample(row[0], masks_to_device(m[:1])[0], gpu(policies[0]), gpu(u[:1]))
    assert host(r.token_ids).tolist() == [int(ref[0])]


def test_offsets_past_32_bits(cuda_lib):
    """Rows more than 2^31 elements apart."""
    rng = np.random.default_rng(21)
    x = normal(rng, (3, 5000), "bf16")
    big = torch.empty((3, 1_200_000_008), dtype=torch.bfloat16, device="cuda")
    view = big[:, :5000]
    view.copy_(to_device(x, "bf16"))
    policies, u = table(POLICIES["all"], 3), rng.random(3)
    r = ox.policy_sample(view, None, gpu(policies), gpu(u))
    np.testing.assert_array_equal(host(r.token_ids),
                                  opol.sample(f64(x, "bf16"), None, policies, u)[0])
    del view, big
    out = torch.empty((3, 800_000_000), dtype=torch.float32, device="cuda")[:, :5000]
    ox.policy_probs(to_device(x, "bf16"), None, gpu(policies), out=out)
    assert_probs(out, opol.probs(f64(x, "bf16"), None, policies)[0])


def test_empty_batches(cuda_lib):
    x = torch.zeros(0, 50, device="cuda")
    pol = torch.zeros(0, 4, dtype=torch.float64, device="cuda")
    r = ox.policy_sample(x, None, pol, torch.zeros(0, device="cuda"))
    assert r.token_ids.shape == (0,) and r.status.shape == (0,)
    p, st = ox.policy_probs(x, None, pol)
    assert p.shape == (0, 50) and st.shape == (0,)
    s = ox.spec_sample(torch.zeros(0, 3, 50, device="cuda"), None,
                       torch.zeros(0, 2, dtype=torch.int32, device="cuda"), pol,
                       torch.zeros(0, 3, device="cuda"))
    assert s.accept_len.shape == (0,)


def test_refusals(cuda_lib):
    x = torch.zeros(2, 64, device="cuda")
    pol = gpu(table(POLICIES["plain"], 2))
    u = torch.zeros(2, device="cuda")
    m = torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    for err, args in (
        (TypeError, (x.double(), None, pol, u)), (TypeError, (x.int(), None, pol, u)),
        (ValueError, (x[None], None, pol, u)), (ValueError, (x[:, :0], None, pol, u)),
        (ValueError, (x, m[:, :1], pol, u)), (ValueError, (x, m[:1], pol, u)),
        (TypeError, (x, m.long(), pol, u)), (TypeError, (x, None, pol.float(), u)),
        (ValueError, (x, None, pol[:1], u)), (ValueError, (x, None, pol[:, :3], u)),
        (ValueError, (x, None, pol.cpu(), u)), (ValueError, (x, None, pol, u[:1])),
        (TypeError, (x, None, pol, u.half())), (ValueError, (x, None, pol, u.cpu())),
        (TypeError, (x, None, [1.0], u)), (ValueError, (x, None, pol, u[:, None])),
    ):
        with pytest.raises(err):
            ox.policy_sample(*args)
    for out in (torch.zeros(2, 63, device="cuda"), torch.zeros(2, 64, device="cuda").double(),
                torch.zeros(1, 64, device="cuda").expand(2, 64), torch.zeros(2, 64),
                torch.zeros(64, 2, device="cuda").t(), x):
        with pytest.raises(ValueError):
            ox.policy_probs(x, None, pol, out=out)
    y = torch.zeros(2, 3, 64, device="cuda")
    d = torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    u = torch.zeros(2, 3, device="cuda")
    for err, args, kw in (
        (ValueError, (y[0], None, d, pol, u), {}), (ValueError, (y[:, :1], None, d, pol, u), {}),
        (TypeError, (y.double(), None, d, pol, u), {}), (ValueError, (y, m, d, pol, u), {}),
        (ValueError, (y, None, d.long(), pol, u), {}), (ValueError, (y, None, d[:, :1], pol, u), {}),
        (ValueError, (y, None, d, pol, u[:, :2]), {}), (ValueError, (y, None, d, pol[:1], u), {}),
        (ValueError, (y, None, d, pol, u), dict(draft_probs=y)),
        (ValueError, (y, None, d, pol, u), dict(draft_probs=y[:, :2].double())),
        (ValueError, (y, None, d, pol, u), dict(draft_lens=d[:, 0].long())),
        (ValueError, (y, None, d, pol, u), dict(draft_lens=d)),
        (ValueError, (y, None, d.cpu(), pol, u), {}),
    ):
        with pytest.raises(err):
            ox.spec_sample(*args, **kw)


def test_same_draw_as_masked_sample(cuda_lib):
    """Temperature and top-p alone, with the numbers masked_sample makes for itself."""
    w = workloads.batched(rows=8)
    x, m = to_device(w["logits_bf16"], "bf16"), masks_to_device(w["masks"])
    for call in range(3):
        u = [osamp.uniform(11, call, r) for r in range(8)]
        a = ox.masked_sample(x, m, temperature=0.8, top_p=0.9, seed=11, call=call)
        pol = ox.pack_policies(ox.SamplingPolicy(temperature=0.8, top_p=0.9))
        b = ox.policy_sample(x, m, pol, gpu(u))
        assert torch.equal(a.token_ids, b.token_ids) and torch.equal(a.status, b.status)


# --------------------------------------------------------------------------------------
# speculative sampling
# --------------------------------------------------------------------------------------
def spec_inputs(rng, batch, gamma, vocab, dtype, masked=True, noise=0.5, temperature=1.0):
    x = rng.standard_normal((batch, gamma + 1, vocab)) * 3
    m = None
    valid = np.ones((batch, gamma, vocab), bool)
    if masked:
        m = workloads.bernoulli_masks(rng, rng.uniform(0.05, 0.6, batch * (gamma + 1)), vocab)
        m = m.reshape(batch, gamma + 1, -1)
        valid = np.stack([[osamp.unpack_mask(m[b, i], vocab) for i in range(gamma)]
                          for b in range(batch)])
    z = x[:, :gamma] + rng.standard_normal((batch, gamma, vocab)) * noise
    z = np.where(valid, z / temperature, -np.inf)
    q = np.exp(z - z.max(-1, keepdims=True))
    q = (q / q.sum(-1, keepdims=True)).astype(np.float32)
    d = np.array([[opol.choose(q[b, i].astype(np.float64), rng.random()) for i in range(gamma)]
                  for b in range(batch)], np.int32)
    return rounded(x, dtype), m, q, d, rng.random((batch, gamma + 1))


def check_spec(x, m, d, policies, u, dtype, q=None, lens=None):
    r = ox.spec_sample(
        to_device(x, dtype), None if m is None else masks_to_device(m), torch.from_numpy(d).cuda(),
        gpu(policies), torch.as_tensor(u).cuda(), draft_probs=None if q is None else
        torch.from_numpy(q).cuda(), draft_lens=None if lens is None else
        torch.as_tensor(lens, dtype=torch.int32).cuda())
    drawn = {}
    taken, token, status = opol.spec(f64(x, dtype), m, d, policies, np.asarray(u, np.float64), q,
                                     lens, drawn)
    np.testing.assert_array_equal(host(r.accept_len), taken)
    got = host(r.correction)
    for b in np.flatnonzero(got != token):
        assert b in drawn and on_boundary(drawn[b], float(u[b, -1]), got[b], token[b]), (
            b, got, token)
    np.testing.assert_array_equal(host(r.status).astype(np.uint32), status)
    return taken


@pytest.mark.parametrize("policy", list(POLICIES))
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_spec_random(dtype, policy, cuda_lib):
    rng = np.random.default_rng(len(dtype) * 1000 + list(POLICIES).index(policy))
    batch, gamma, vocab = 7, 4, 2003
    t = POLICIES[policy][0] or 0.3
    for masked in (True, False):
        x, m, q, d, u = spec_inputs(rng, batch, gamma, vocab, dtype, masked, temperature=t)
        pol = table(POLICIES[policy], batch)
        check_spec(x, m, d, pol, u, dtype, q)
        check_spec(x, m, d, pol, u.astype(np.float32), dtype, None)
        lens = rng.integers(0, gamma + 1, batch)
        check_spec(x, m, d, pol, u, dtype, q, lens)


def test_spec_accepts_and_refuses(cuda_lib):
    """A draft model near the target: every accepted length occurs, 0 to gamma."""
    rng = np.random.default_rng(2)
    x, m, q, d, u = spec_inputs(rng, 60, 3, 801, "f32", noise=0.7)
    taken = check_spec(x, m, d, table(POLICIES["plain"], 60), u, "f32", q)
    assert set(taken.tolist()) == {0, 1, 2, 3}


@pytest.mark.parametrize("batch,gamma,vocab", [(1, 1, 5), (1, 1, 40000), (1, 7, 20000),
                                               (3, 255, 70), (150, 1, 300), (40, 4, 9001),
                                               (500, 3, 700)])
def test_spec_shapes(batch, gamma, vocab, cuda_lib):
    rng = np.random.default_rng(batch * 1000 + gamma)
    x, m, q, d, u = spec_inputs(rng, batch, gamma, vocab, "bf16", noise=0.1)
    names = list(POLICIES)
    policies = np.stack([POLICIES[names[i]] for i in rng.integers(0, len(names), batch)])
    policies[:, 0] = np.where(policies[:, 0] == 0, 0, 1.0)
    check_spec(x, m, d, policies, u, "bf16", q)
    check_spec(x, None, d, policies, u, "bf16", q)


def test_spec_special_rows(cuda_lib):
    rng = np.random.default_rng(31)
    x, m, q, d, u = spec_inputs(rng, 14, 3, 500, "f32", noise=0.0)
    u[:, :3] = 0.01  # every draft accepted, unless the row says otherwise
    lens = np.full(14, 3)
    m[0, 0] = 0                      # no valid id at the first row
    x[1, 2] = np.nan                 # a bad row behind two accepted drafts
    x[2, 3, :] = -np.inf             # the row after the last draft
    x[3, 1, :] = np.nan
    u[3, 0] = 1.0 - 2.0**-53         # refused before the bad row is reached
    q[3, 0, d[3, 0]] = 1.0
    lens[4], lens[5] = -1, 4         # lengths outside [0, gamma]
    u[6, 3] = 1.0                    # the drawing number outside [0, 1)
    u[7, 1] = np.nan
    d[8, 1] = 500                    # drafts outside the vocabulary
    d[9, 0] = -3
    q[10, 0] = np.nan                # probabilities that are none
    q[11, 0] = -1.0
    q[12, 0] = 2.0                   # nothing remains: the draw is from p
    u[12, 0] = 0.9
    x[13, 0, :] = 0.0
    x[13, 0, d[13, 0]] = np.inf
    m[13, 0] = 0xFFFFFFFF
    check_spec(x, m, d, table(POLICIES["plain"], 14), u, "f32", q, lens)
    check_spec(x, m, d, table(POLICIES["all"], 14), u, "f32", q, lens)
    check_spec(x, m, d, table(POLICIES["plain"], 14), u, "f32", None, lens)
    bad = table(POLICIES["plain"], 14)
    bad[5:8, 2] = 0.0
    check_spec(x, m, d, bad, u, "f32", q, lens)


def test_spec_ties_at_the_cut(cuda_lib):
    """A draft that ties with the cut is kept or not by its place among the ties."""
    x = np.zeros((6, 2, 3000), np.float32)
    x[:, :, 2000:] = -1.0
    d = np.array([[0], [99], [100], [101], [1999], [2500]], np.int32)
    q = np.full((6, 1, 3000), 1.0 / 3000, np.float32)
    for k in (100, 101, 2000):
        for u0 in (0.0, 0.05, 0.9):
            u = np.full((6, 2), 0.37)
            u[:, 0] = u0
            check_spec(x, None, d, table((1.0, k, 1.0, 0.0), 6), u, "f32", q)
            check_spec(x, None, d, table((1.0, k, 1.0, 0.0), 6), u, "f32", None)


def test_spec_strides(cuda_lib):
    rng = np.random.default_rng(14)
    x, m, q, d, u = spec_inputs(rng, 5, 3, 1999, "bf16")
    pol = table(POLICIES["all"], 5)
    ref = opol.spec(f64(x, "bf16"), m, d, pol, u, q)
    xt = torch.zeros(6, 5, 2050, dtype=torch.bfloat16, device="cuda")
    xt[1:, :4, 7:2006] = to_device(x, "bf16")
    qt = torch.zeros(5, 4, 2001, device="cuda")
    qt[:, 1:, 1:2000] = torch.from_numpy(q).cuda()
    mt = torch.zeros(5, 5, m.shape[2] + 3, dtype=torch.int32, device="cuda")
    mt[:, 1:, : m.shape[2]] = masks_to_device(m)
    dt = torch.zeros(5, 9, dtype=torch.int32, device="cuda")
    dt[:, 2:8:2] = torch.from_numpy(d).cuda()
    ut = torch.zeros(4, 5, dtype=torch.float64, device="cuda")
    ut.copy_(torch.from_numpy(u).t())
    r = ox.spec_sample(xt[1:, :4, 7:2006], mt[:, 1:], dt[:, 2:8:2], gpu(pol), ut.t(),
                       draft_probs=qt[:, 1:, 1:2000])
    for got, want in zip((r.accept_len, r.correction, r.status), ref):
        np.testing.assert_array_equal(host(got).astype(np.int64), want.astype(np.int64))


# --------------------------------------------------------------------------------------
# a run of them together, streams and graphs
# --------------------------------------------------------------------------------------
def test_speculative_step_together(cuda_lib):
    """Draft with policy_probs and policy_sample, verify with spec_sample, as one step."""
    rng = np.random.default_rng(40)
    batch, gamma, vocab = 9, 3, 12000
    target = normal(rng, (batch, gamma + 1, vocab), "bf16")
    draft = rounded(f64(target[:, :gamma], "bf16") + rng.standard_normal(
        (batch, gamma, vocab)) * 0.3, "bf16")
    m = workloads.bernoulli_masks(rng, rng.uniform(0.02, 0.3, batch * (gamma + 1)), vocab)
    m = m.reshape(batch, gamma + 1, -1)
    names = [n for n in POLICIES if n not in ("top_p_small", "min_p_all")]
    policies = np.stack([POLICIES[names[b % len(names)]] for b in range(batch)])
    u_draft, u = rng.random((batch, gamma)), rng.random((batch, gamma + 1))
    pol = ox.pack_policies([ox.SamplingPolicy(float(t), int(k), float(p), float(mp))
                            for t, k, p, mp in policies])
    xd, mt = to_device(draft, "bf16"), masks_to_device(m)
    q = torch.empty(batch, gamma, vocab, device="cuda")
    drafts = torch.empty(batch, gamma, dtype=torch.int32, device="cuda")
    for i in range(gamma):
        ox.policy_probs(xd[:, i], mt[:, i], pol, out=q[:, i])
        drafts[:, i] = ox.policy_sample(xd[:, i], mt[:, i], pol, gpu(u_draft[:, i])).token_ids
    for i in range(gamma):
        ids, _ = opol.sample(f64(draft[:, i], "bf16"), m[:, i], policies, u_draft[:, i])
        np.testing.assert_array_equal(host(drafts[:, i]), ids)
        assert_probs(q[:, i], opol.probs(f64(draft[:, i], "bf16"), m[:, i], policies)[0])
    r = ox.spec_sample(to_device(target, "bf16"), mt, drafts, pol, gpu(u), draft_probs=q)
    ref = opol.spec(f64(target, "bf16"), m, host(drafts), policies, u, host(q))
    for got, want in zip((r.accept_len, r.correction, r.status), ref):
        np.testing.assert_array_equal(host(got).astype(np.int64), want.astype(np.int64))


def test_streams_and_graph_replay(cuda_lib):
    """Captured calls replay on changed logits, policies and numbers, beside eager calls on
    another stream."""
    rng = np.random.default_rng(50)
    batch, gamma, vocab = 4, 2, 30011
    sets = []
    for i in range(3):
        x, m, q, d, u = spec_inputs(rng, batch, gamma, vocab, "bf16", noise=0.2)
        policies = np.stack([POLICIES[n] for n in (("top_p", "all", "plain", "top_k"),
                                                   ("min_p", "greedy", "all", "top_p"),
                                                   ("k_wide", "top_p", "greedy", "plain"))[i]])
        sets.append((to_device(x, "bf16"), masks_to_device(m), torch.from_numpy(q).cuda(),
                     torch.from_numpy(d).cuda(), gpu(u), gpu(policies)))

    def run(x, m, q, d, u, pol):
        a = ox.policy_sample(x[:, 0], m[:, 0], pol, u[:, 0])
        p, st = ox.policy_probs(x[:, 1], m[:, 1], pol)
        s = ox.spec_sample(x, m, d, pol, u, draft_probs=q)
        return [a.token_ids, a.status, p, st, s.accept_len, s.correction, s.status]

    eager = [[t.clone() for t in run(*s)] for s in sets]
    static = [t.clone() for t in sets[0]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(*static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run(*static)
    for i in (1, 2, 0, 1):
        for t, new in zip(static, sets[i]):
            t.copy_(new)
        torch.cuda.synchronize()
        side.wait_stream(torch.cuda.current_stream())
        graph.replay()
        with torch.cuda.stream(side):
            other = run(*sets[2])
        torch.cuda.synchronize()
        for got, want in zip(held, eager[i]):
            assert torch.equal(got, want)
        for got, want in zip(other, eager[2]):
            assert torch.equal(got, want)


def test_calls_at_once_on_two_streams(cuda_lib):
    """Each call has a workspace of its own, so calls on two streams may overlap."""
    rng = np.random.default_rng(55)
    x, m, q, d, u = spec_inputs(rng, 6, 3, 40009, "f16", noise=0.2)
    pol = gpu(np.stack([POLICIES[n] for n in ("top_p", "all", "plain", "top_k", "greedy",
                                              "min_p")]))
    args = (to_device(x, "f16"), masks_to_device(m), torch.from_numpy(d).cuda(), pol, gpu(u))
    qt = torch.from_numpy(q).cuda()
    want = ox.spec_sample(*args, draft_probs=qt)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(ox.spec_sample(*args, draft_probs=qt))
    torch.cuda.synchronize()
    for r in got:
        for a, b in zip((r.accept_len, r.correction, r.status),
                        (want.accept_len, want.correction, want.status)):
            assert torch.equal(a, b)


def test_repeated_calls_give_the_same_bits(cuda_lib):
    rng = np.random.default_rng(60)
    x = to_device(normal(rng, (20, 50021), "f32"), "f32")
    pol = gpu(table((1.1, 0, 0.97, 0.0), 20))
    first = ox.policy_probs(x, None, pol)[0].clone()
    for _ in range(5):
        assert torch.equal(ox.policy_probs(x, None, pol)[0], first)


def test_probs_refuses_outputs_over_its_inputs(cuda_lib):
    x = torch.zeros(2, 64, device="cuda")
    pol = gpu(table((1.0, 0, 1.0, 0.0), 2))
    words = torch.full((130,), -1, dtype=torch.int32, device="cuda")
    over_mask = words.view(torch.float32)[:128].view(2, 64)
    with pytest.raises(ValueError):
        ox.policy_probs(x, words[:4].view(2, 2), pol, out=over_mask)
    over_policies = torch.zeros(64, dtype=torch.float64, device="cuda")
    with pytest.raises(ValueError):
        ox.policy_probs(x, None, over_policies[:8].view(2, 4),
                        out=over_policies.view(torch.float32).view(2, 64))
    with pytest.raises(ValueError):
        ox.policy_probs(x, None, pol, out=x)


def test_lengths_out_of_range_in_a_batch_of_several_launches(cuda_lib):
    """More rows than one launch takes: every entry's later rows look at what the earlier ones
    decided, and a length may be anything that 32 bits hold."""
    batch, gamma, vocab = 300, 3, 500
    rng = np.random.default_rng(61)
    x = to_device(normal(rng, (batch * (gamma + 1), vocab), "f32"), "f32")
    x = x.view(batch, gamma + 1, vocab)
    d = torch.from_numpy(rng.integers(0, vocab, (batch, gamma)).astype(np.int32)).cuda()
    lens = torch.from_numpy(rng.integers(0, gamma + 1, batch).astype(np.int32))
    bad = {0: 2**31 - 1, 7: -(2**31), 150: -1, 299: gamma + 1}
    for i, n in bad.items():
        lens[i] = n
    pol = gpu(table((1.0, 0, 0.9, 0.0), batch))
    u = gpu(rng.random((batch, gamma + 1)))
    r = ox.spec_sample(x, None, d, pol, u, draft_lens=lens.cuda())
    status = r.status.cpu().numpy()
    for i in range(batch):
        assert status[i] == (ox.STATUS_BAD_POLICY if i in bad else 0)
    assert (r.correction.cpu().numpy()[list(bad)] == -1).all()
    assert (r.accept_len.cpu().numpy()[list(bad)] == 0).all()


@pytest.mark.parametrize("dtype", ("f32", "f16", "bf16"))
@pytest.mark.parametrize("scale", (20.0, 45.0, 400.0))
@pytest.mark.parametrize("rows,vocab", ((1, 20011), (24, 100003), (3, 700)))
def test_peaked_rows(cuda_lib, rows, vocab, scale, dtype):
    """Logits far above the temperature: the maximum lies past the bins, and a few ids among
    the largest peaks hold the mass; also with many of them tied, and under masks."""
    rng = np.random.default_rng(int(scale) + vocab)
    v = rng.standard_normal((rows, vocab)) * scale
    v[:, 3] += scale  # a maximum far above the others
    v[rows // 2, 5:900:2] = v[rows // 2].max()  # equal ones, more than fit the short list
    x = rounded(v, dtype)
    m = workloads.bernoulli_masks(rng, rng.uniform(0.05, 0.9, rows), vocab)
    u = rng.random(rows)
    for policy in ((1.0, 0, 0.9, 0.0), (0.1, 0, 0.95, 0.02), (1.3, 40, 0.99, 0.0),
                   (8.0, 0, 0.7, 0.0), (1.0, 2000, 0.97, 0.0)):
        check(x, None, dtype, table(policy, rows), u)
        check(x, m, dtype, table(policy, rows), u)


# --------------------------------------------------------------------------------------
# rows that stream through a ring of slots, over which the lists of later passes lie
# --------------------------------------------------------------------------------------
RING = {  # rows, vocabulary, views of a row padded by so many ids, mask
    "masked_64": (64, 128256, 0, True), "one_cta_256": (256, 32000, 0, False),
    "one_cta_masked": (300, 33333, 5, True), "odd_64": (64, 151665, 3, False),
    "one_row": (1, 300007, 0, True), "large_256": (256, 128256, 0, False),
}
RING_POLICIES = ("greedy", "min_p", "top_p", "top_k", "plain", "all")


def assert_ring(rows, vocab, dtype, masked):
    code = {"f32": _lib.DTYPE_F32, "f16": _lib.DTYPE_F16, "bf16": _lib.DTYPE_BF16}[dtype]
    out = (ctypes.c_int32 * 5)()
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert _lib.load().onyx_policy_layout(rows, vocab, code, int(masked), sms, out) == _lib.OK
    assert out[2] and not out[3], "these rows are kept whole: the case tests something else"


def ring_rows(rows, vocab, pad, masked, dtype, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    full = torch.randn(rows, vocab + pad, generator=gen, device="cuda").mul_(3.0)
    x = full.to({"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dtype])
    m = None
    if masked:  # from half of the ids down to one in 64
        words = torch.full((rows, (vocab + 31) // 32), -1, dtype=torch.int32, device="cuda")
        depth = torch.arange(rows, device="cuda").view(-1, 1) % 6
        for i in range(6):
            more = torch.randint(-2**31, 2**31, words.shape, generator=gen, device="cuda",
                                 dtype=torch.int32)
            words = torch.where(depth >= i, words & more, words)
        m = words
    u = torch.rand(rows, generator=gen, device="cuda", dtype=torch.float64)
    return x[:, :vocab], m, u


def oracle_row(x, m, policy, u, got):
    """One row on the host: whether `got` is the draw."""
    v = x.float().cpu().numpy().astype(np.float64)
    valid = np.ones(v.size, bool) if m is None else osamp.unpack_mask(
        host(m).view(np.uint32), v.size)
    status, w = opol.kept_weights(v, valid, policy)
    assert status == 0
    want = opol.choose(w, u)
    assert got == want or on_boundary(w, u, got, want), (policy, got, want)
    return w


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("shape", list(RING))
def test_ring_rows(shape, dtype, cuda_lib):
    """Policies mixed over a batch, against the oracle; then the same call again, which gives
    the same draws, alone and while another stream keeps memory busy."""
    rows, vocab, pad, masked = RING[shape]
    assert_ring(rows, vocab, dtype, masked)
    x, m, u = ring_rows(rows, vocab, pad, masked, dtype, rows + vocab)
    policies = np.stack([POLICIES[RING_POLICIES[r % 6]] for r in range(rows)])
    pol = gpu(policies)
    first = ox.policy_sample(x, m, pol, u)
    assert not first.status.any()
    probs, status = ox.policy_probs(x, m, pol)
    assert not status.any()
    some = sorted({0, rows - 1, *range(min(rows, 6)), *range(rows // 2, min(rows, rows // 2 + 6))})
    ids, numbers = host(first.token_ids), host(u)
    for r in some:
        w = oracle_row(x[r], None if m is None else m[r], policies[r], numbers[r], ids[r])
        assert_probs(probs[r], w / w.sum())
    side, junk = torch.cuda.Stream(), torch.empty(1 << 28, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    again = []
    for i in range(16):
        if i >= 8:
            with torch.cuda.stream(side):
                junk.add_(1)
        again.append(ox.policy_sample(x, m, pol, u))
    p = ox.policy_probs(x, m, pol)[0]
    torch.cuda.synchronize()
    for a in again:
        assert torch.equal(a.token_ids, first.token_ids) and torch.equal(a.status, first.status)
    assert torch.equal(p, probs)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("shape", list(RING))
def test_ring_rows_greedy(shape, dtype, cuda_lib):
    """A whole batch at temperature 0, where the least lies between the first pass and the
    lists: the ids of masked_argmax, every time."""
    rows, vocab, pad, masked = RING[shape]
    x, m, u = ring_rows(rows, vocab, pad, masked, dtype, rows * 3 + vocab)
    want = ox.masked_argmax(x, m).token_ids
    pol = gpu((0.0, 0, 1.0, 0.0))
    got = [ox.policy_sample(x, m, pol, u) for _ in range(24)]
    for g in got:
        assert torch.equal(g.token_ids, want) and not g.status.any()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_ring_rows_min_p_alone(dtype, cuda_lib):
    """min-p without another cut: no histogram, the lists follow the first pass at once."""
    rows, vocab, pad, masked = RING["masked_64"]
    x, m, u = ring_rows(rows, vocab, pad, masked, dtype, 17)
    policy = (1.0, 0, 1.0, 0.02)
    got = [ox.policy_sample(x, m, gpu(policy), u).token_ids for _ in range(24)]
    for g in got:
        assert torch.equal(g, got[0])
    for r in range(0, rows, 9):
        oracle_row(x[r], m[r], policy, host(u)[r], host(got[0])[r])


@pytest.mark.parametrize("with_q", [True, False])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_ring_spec(dtype, with_q, cuda_lib):
    """A speculative batch of 32 x 5 rows under every policy, against the oracle."""
    batch, gamma, vocab = 32, 4, 151936
    rows = batch * (gamma + 1)
    assert_ring(batch * (gamma + 1), vocab, dtype, True)
    x, m, _ = ring_rows(rows, vocab, 0, True, dtype, 5 + with_q)
    x, m = x.view(batch, gamma + 1, vocab), m.view(batch, gamma + 1, -1)
    policies = np.stack([POLICIES[RING_POLICIES[b % 6]] for b in range(batch)])
    pol = gpu(policies)
    gen = torch.Generator(device="cuda").manual_seed(9)
    q = torch.empty(batch, gamma, vocab, device="cuda")
    d = torch.empty(batch, gamma, dtype=torch.int32, device="cuda")
    for i in range(gamma):
        near = (x[:, i].float() + 0.3 * torch.randn(batch, vocab, generator=gen, device="cuda")
                ).to(x.dtype)
        ox.policy_probs(near, m[:, i], pol, out=q[:, i])
        u = torch.rand(batch, generator=gen, device="cuda", dtype=torch.float64)
        d[:, i] = ox.policy_sample(near, m[:, i], pol, u).token_ids
    u = torch.rand(batch, gamma + 1, generator=gen, device="cuda", dtype=torch.float64)
    q = q if with_q else None
    first = ox.spec_sample(x, m, d, pol, u, draft_probs=q)
    again = [ox.spec_sample(x, m, d, pol, u, draft_probs=q) for _ in range(8)]
    for a in again:
        for got, want in zip((a.accept_len, a.correction, a.status),
                             (first.accept_len, first.correction, first.status)):
            assert torch.equal(got, want)
    taken, token = host(first.accept_len), host(first.correction)
    assert not first.status.any()
    for b in range(0, batch, 3):
        drawn = {}
        want = opol.spec(x[b:b + 1].float().cpu().numpy().astype(np.float64),
                         host(m[b:b + 1]).view(np.uint32), host(d[b:b + 1]), policies[b:b + 1],
                         host(u[b:b + 1]), None if q is None else host(q[b:b + 1]), None, drawn)
        assert taken[b] == want[0][0]
        if token[b] != want[1][0]:
            assert on_boundary(drawn[0], float(u[b, -1]), token[b], want[1][0])


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("temperature", [1e30, 6e35, 1e37, 1e300, 1.7e308])
def test_very_high_temperatures(temperature, dtype, cuda_lib):
    """Every finite value weighs 1 there, and a logit of -inf still nothing."""
    rng = np.random.default_rng(101)
    x = rng.standard_normal((5, 5003)) * 3
    x[1, rng.random(5003) < 0.4] = -np.inf
    x[2, 1::2] = -np.inf
    x[3, :5000] = -np.inf
    x[4, 0] = -np.inf
    x = rounded(x, dtype)
    m = workloads.bernoulli_masks(rng, np.full(5, 0.5), 5003)
    m[:, 0] |= np.uint32(3)
    m[:, -1] |= np.uint32(1 << 10)
    for policy in ((temperature, 0, 1.0, 0.0), (temperature, 0, 0.77123, 0.0),
                   (temperature, 700, 0.5123, 0.0), (temperature, 0, 1.0, 0.3)):
        check(x, None, dtype, table(policy, 5), rng.random(5))
        check(x, m, dtype, table(policy, 5), rng.random(5))


@pytest.mark.parametrize("policy", [(1.0, 0, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (1.3, 0, 1.0, 0.0)])
def test_values_of_ten_billion_temperatures(policy, cuda_lib):
    """float32 values whose spacing is wider than the range of weights that are summed: the
    next value below the largest weighs nothing."""
    rng = np.random.default_rng(102)
    x = (1.1e10 + 1024.0 * rng.integers(-4, 4, (6, 7001))).astype(np.float32)
    x[3] = -x[3]
    x[4] = np.float32(1.7e10) + 1024.0 * rng.integers(-2, 1, 7001)
    x[5, 4000:] = np.float32(2.0**33)
    check(x, None, "f32", table(policy, 6), rng.random(6))
    m = workloads.bernoulli_masks(rng, np.full(6, 0.5), 7001)
    check(x, m, "f32", table(policy, 6), rng.random(6))


def raw_sample(x, m, dtype, policies, u):
    """policy_sample by its C entry, into outputs that hold -7: a row that nothing is written
    for shows."""
    xt, mt = to_device(x, dtype), None if m is None else masks_to_device(m)
    pol, ut = gpu(policies), gpu(u)
    rows, vocab = xt.shape
    ids = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    status = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    code = {"f32": _lib.DTYPE_F32, "f16": _lib.DTYPE_F16, "bf16": _lib.DTYPE_BF16}[dtype]
    _lib.check("onyx_policy_sample", _lib.load().onyx_policy_sample(
        xt.data_ptr(), code, rows, vocab, vocab, None if mt is None else mt.data_ptr(),
        0 if mt is None else mt.stride(0), pol.data_ptr(), 4, ut.data_ptr(), _lib.DTYPE_F64, 1,
        ids.data_ptr(), status.data_ptr(), torch.cuda.current_stream().cuda_stream))
    return host(ids), host(status)


@pytest.mark.parametrize("dtype,high,t,low", [("f32", 619.0, 1.0, -32.0), ("f16", 619.0, 1.0, -32.0),
                                              ("bf16", 500.0, 0.81, -27.0),
                                              ("f32", 700.0, 1.0, -32.0),
                                              ("f32", 560.0, 1.0, -32.0)])
def test_masked_ids_far_above_the_valid_ones(dtype, high, t, low, cuda_lib):
    """Ids that the mask takes out, hundreds of T above the rest, at the places that the kernel
    samples: what is summed relative to them must still hold the valid ids' small weights.
    n of these, of weight w, follow the largest one (weight 1), and u lies in their share. The
    draw is the one whose rank passes (u (1 + n w) - 1) / w. Two sums of n weights, each within
    n 2^-53 of its value, decide it, and as many the cut that top-p makes: 4 n 2^-53 / w ranks."""
    vocab = 200000
    x = np.full((2, vocab), low)
    x[:, 1] = 0.0
    at = np.arange(128) * vocab >> 7
    x[:, at] = high
    valid = np.ones(vocab, bool)
    valid[at] = False
    words = np.packbits(np.pad(valid, (0, -vocab % 32)), bitorder="little").view(np.uint32)
    valid[1] = False
    lows, w = np.flatnonzero(valid), math.exp(low / t)
    n = lows.size
    for p in (1.0, 1.0 - n * w * 0.02):
        kept = n if p == 1.0 else math.ceil((p - 1.0 + p * n * w) / w)
        u = np.array([1.0 - n * w * 0.5, 1.0 - n * w * 0.1])
        ids, status = raw_sample(rounded(x, dtype), np.stack([words, words]), dtype,
                                 table((t, 0, p, 0.0), 2), u)
        assert (status == 0).all()
        want = (u - 1.0 + u * kept * w) / w
        assert np.isin(ids, lows).all(), ids
        assert (np.abs(np.searchsorted(lows, ids) - want) <= 4 * n * 2.0**-53 / w + 2).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_weights_that_underflow_are_not_drawn(dtype, cuda_lib):
    """Weights below 2^-1000 count as 0. The largest value lies far above those that the first
    pass measures by; the parts of the row before it hold ids that weigh nothing."""
    vocab = 40000
    x = np.zeros((4, vocab))
    x[:, :5000] = -550.0
    x[:, 20001] = 160.0
    x[:, 39000:] = -550.0
    x[1, :5000] = -540.0     # 700 T below
    x[2, :5000] = -530.0     # 690 T below: 2^-995
    x[3, 20001] = 100.0
    x = rounded(x, dtype)
    v = f64(x, dtype)
    u = np.array([0.0, 1e-320, 2.0**-400, 1.0 - 2.0**-53])
    for ui in u:
        ids, status = raw_sample(x, None, dtype, table((1.0, 0, 1.0, 0.0), 4), np.full(4, ui))
        assert (status == 0).all()
        for r in range(4):
            w = np.exp(v[r] - v[r].max())
            w[w < 2.0**-1000] = 0.0
            assert ids[r] == opol.choose(w, ui), (r, ui)


def test_min_p_at_the_weight_of_the_cut(cuda_lib):
    """min_p next to the weight of the value that top-k cuts at, which lies in a part of the row
    of its own: that id is kept or not, and in either case something is drawn."""
    vocab, top = 9001, 8000
    rows, policies = [], []
    for j in range(1, 161):
        low = 10.0 - j / 16.0
        w = math.exp(low - 10.0)
        for steps in range(-4, 5):
            row = np.full(vocab, -100.0)
            row[[0, 1, top]] = low, low, 10.0
            rows.append(row)
            policies.append((1.0, 2, 0.9999999, w * (1.0 + steps * 2.0**-52)))
    policies = np.array(policies)
    x = rounded(np.stack(rows), "bf16")
    for dtype, values in (("bf16", x), ("f32", f64(x, "bf16").astype(np.float32))):
        ids, status = raw_sample(values, None, dtype, policies, np.zeros(len(rows)))
        assert (status == 0).all()
        assert np.isin(ids, (0, top)).all()
        p, st = ox.policy_probs(to_device(values, dtype), None, gpu(policies))
        p = host(p).astype(np.float64)
        assert not host(st).any()
        # what is drawn at u = 0 is what has a probability, and they sum to 1
        np.testing.assert_array_equal(np.where(p[:, 0] > 0, 0, top), ids)
        assert (np.abs(p.sum(1) - 1.0) <= 2.0**-23).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("lows", [1, 3, 8])
def test_min_p_at_the_weight_of_an_id(lows, dtype, cuda_lib):
    """min_p next to the weight of ids that have a part of the row to themselves: the passes that
    sum and the one that draws agree on whether they are kept, one to a lane or many."""
    vocab, top = 9001, 8000
    rows, weights = [], []
    for j in range(1, 161):
        low = 10.0 - j / 16.0
        w = math.exp(low - 10.0)
        for steps in range(-6, 7):
            row = np.full(vocab, -100.0)
            row[:lows], row[top] = low, 10.0
            rows.append(row)
            weights.append(w * (1.0 + steps * 2.0**-52))
    values, n = rounded(np.stack(rows), dtype), len(rows)
    for k, p in ((0, 1.0), (0, 0.9999999), (20, 1.0), (600, 0.9999999)):
        policies = np.stack([np.ones(n), np.full(n, k), np.full(n, p), weights], axis=1)
        ids, status = raw_sample(values, None, dtype, policies, np.zeros(n))
        assert (status == 0).all() and np.isin(ids, (0, top)).all()
        probs, st = ox.policy_probs(to_device(values, dtype), None, gpu(policies))
        probs = host(probs).astype(np.float64)
        assert not host(st).any()
        np.testing.assert_array_equal(np.where(probs[:, 0] > 0, 0, top), ids)
        # each of the 9 probabilities at most is rounded by 2^-24 of itself
        assert (np.abs(probs.sum(1) - 1.0) <= 2.0**-23).all()


def test_probs_beside_the_logits_in_one_buffer(cuda_lib):
    """Logits and probabilities as two columns of one float32 buffer share no memory."""
    rng = np.random.default_rng(111)
    x = normal(rng, (6, 3001), "f32")
    both = torch.full((6, 2, 3010), 7.0, device="cuda")
    both[:, 0, :3001] = to_device(x, "f32")
    policies = table(POLICIES["all"], 6)
    p, status = ox.policy_probs(both[:, 0, :3001], None, gpu(policies), out=both[:, 1, 4:3005])
    assert not status.any()
    assert_probs(p, opol.probs(f64(x, "f32"), None, policies)[0])
    np.testing.assert_array_equal(host(both[:, 0, :3001]), x)
    assert (host(both[:, 0, 3001:]) == 7).all() and (host(both[:, 1, :4]) == 7).all()
    assert (host(both[:, 1, 3005:]) == 7).all()
    with pytest.raises(ValueError, match="share memory"):
        ox.policy_probs(both[:, 0, :3001], None, gpu(policies), out=both.view(6, -1)[:, 3000:6001])


# --------------------------------------------------------------------------------------
# the accuracy of a weight
# --------------------------------------------------------------------------------------
def weight_by_bisection(low, top, dtype, policy):
    """The largest u at which id 0 of the row [low, top] is drawn, for every `low`: the kernel
    draws it while w > u (w + 1), so u = w / (w + 1). Bits of float64 numbers are halved."""
    values = rounded(np.stack([low, np.full(low.size, top)], axis=1), dtype)
    x, pol = to_device(values, dtype), gpu(policy)
    lo = torch.zeros(low.size, dtype=torch.int64, device="cuda")
    hi = torch.full_like(lo, int(np.float64(0.75).view(np.int64)))
    for _ in range(63):
        mid = lo + (hi - lo) // 2
        r = ox.policy_sample(x, None, pol, mid.view(torch.float64))
        drawn = r.token_ids == 0
        lo, hi = torch.where(drawn, mid, lo), torch.where(drawn, hi, mid)
    assert (hi - lo <= 1).all()
    return f64(values, dtype)[:, 0], host(lo.view(torch.float64))


def weight_error(low, top, t, u):
    """For every id x = (low - top) / t and the relative distance of u from w / (w + 1), w = exp(x),
    with 40 digits."""
    with decimal.localcontext() as ctx:
        ctx.prec = 40
        for a, b in zip(low.tolist(), u.tolist()):
            x = (decimal.Decimal(a) - decimal.Decimal(top)) / decimal.Decimal(t)
            w = x.exp()
            yield float(x), float(decimal.Decimal(b) * (w + 1) / w - 1)


@pytest.mark.parametrize("t", [1.0, 0.7, 3.3, 0.01])
def test_accuracy_of_a_weight(t, cuda_lib):
    """exp2_table() is within 2^-50. Its argument (v - max) log2(e) 16 / T is rounded by four
    operations (1 / T, the constant, their product, the last product), each by 2^-53 of it: a
    relative error of |x| 4 2^-53 of w = exp(x). The sum w + 1, its product with u and the last
    place of u add 4 2^-53."""
    rng = np.random.default_rng(120)
    low = -rng.uniform(0.0, 690.0 * t, 2000)
    low[:400] = -rng.uniform(0.0, 2.0 * t, 400)
    low, u = weight_by_bisection(low, 0.0, "f32", (t, 0, 1.0, 1e-305))
    for x, err in weight_error(low, 0.0, t, u):
        assert abs(err) <= 2.0**-50 + abs(x) * 2.0**-51 + 2.0**-51, (x, err * 2.0**50)


@pytest.mark.parametrize("t", [1.0, 0.7, 1.3])
def test_accuracy_of_a_weight_from_the_table(t, cuda_lib):
    """bfloat16 rows under top-p: a weight is the first of 8 times a ratio up to 7 times, each of
    the eight factors within 2^-50 and their products rounded: 2^-47 + 7 2^-53, beside the
    argument's part and 4 2^-53 for the sum, the product and u."""
    low = 10.0 - np.arange(1, int(15 * t * 16)) / 16.0
    low, u = weight_by_bisection(low, 10.0, "bf16", (t, 0, 0.9999999, 0.0))
    for x, err in weight_error(low, 10.0, t, u):
        assert abs(err) <= 2.0**-47 + abs(x) * 2.0**-51 + 11 * 2.0**-53, (x, err * 2.0**50)


# --------------------------------------------------------------------------------------
# the largest sizes
# --------------------------------------------------------------------------------------
@pytest.mark.parametrize("vocab", [1 << 30, (1 << 30) - 5])
def test_longest_rows(vocab, cuda_lib):
    """The longest row, whole and from an odd offset: the first maximum, the first k of the
    ranking, and draws by float64 sums of pieces. Two sums of n weights decide a draw, each
    within n 2^-53 of its value: the mass up to the id drawn is within 2 n 2^-53 of u times the
    total, but for that id's own weight."""
    gen = torch.Generator(device="cuda").manual_seed(7)
    x = torch.empty(1, 1 << 30, dtype=torch.bfloat16, device="cuda")
    for part in x[0].split(1 << 27):
        part.copy_(torch.randn(part.numel(), generator=gen, device="cuda").mul_(3.0))
    x = x[:, (1 << 30) - vocab:]
    top = x.max()
    pol = gpu((0.0, 0, 1.0, 0.0))
    half = torch.full((1,), 0.5, dtype=torch.float64, device="cuda")
    want = int((x[0] == top).nonzero()[0])
    assert int(ox.policy_sample(x, None, pol, half).token_ids) == want
    # the first three of the ranking: values falling, ids rising among equals
    levels = torch.cat([p.topk(3)[0] for p in x[0].split(1 << 27)]).sort(descending=True)[0][:3]
    some = (x[0] >= levels[-1]).nonzero().squeeze(1)
    first = sorted(some.tolist(), key=lambda i: (-float(x[0, i]), i))[:3]
    got = [int(ox.policy_sample(x, None, gpu((1.0, 3, 1.0, 0.0)),
                                torch.tensor([u], device="cuda")).token_ids)
           for u in (0.0, 0.5, 1.0 - 2.0**-24)]
    assert set(got) <= set(first) and got[0] == min(first) and got[-1] == max(first)
    masses = torch.stack([torch.exp(p.double() - top.double()).sum()
                          for p in x[0].split(1 << 24)]).cumsum(0)
    for u in (1e-9, 0.37, 0.9999):
        r = ox.policy_sample(x, None, gpu((1.0, 0, 1.0, 0.0)), half * 0 + u)
        at = int(r.token_ids)
        assert not r.status.any() and 0 <= at < vocab
        piece = at >> 24
        w = torch.exp(x[0, piece << 24: at + 1].double() - top.double())
        through = float(w.sum()) + (float(masses[piece - 1]) if piece else 0.0)
        total = float(masses[-1])
        slack = 2 * vocab * 2.0**-53 * total
        assert through - float(w[-1]) - slack <= u * total <= through + slack


def test_many_short_rows(cuda_lib):
    """More rows than 16 bits count, of 3 ids each."""
    rng = np.random.default_rng(130)
    rows = 70001
    x = normal(rng, (rows, 3), "f32")
    policies = np.stack([POLICIES[n] for n in ("plain", "greedy", "top_k1", "top_p", "min_p")])
    policies = policies[np.arange(rows) % 5]
    u = rng.random(rows)
    ids, status = raw_sample(x, None, "f32", policies, u)
    assert (status == 0).all()
    some = np.concatenate([np.arange(500), np.arange(rows - 500, rows)])
    want = opol.sample(f64(x[some], "f32"), None, policies[some], u[some])[0]
    np.testing.assert_array_equal(ids[some], want)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_min_p_where_weights_round_to_equal(dtype, cuda_lib):
    """min_p keeps the ids whose float64 weight reaches it: values that differ by less than
    2^-56 T weigh exactly 1, as the largest does."""
    rng = np.random.default_rng(140)
    x = rng.standard_normal((4, 5003)) * 3
    x[1, ::3] = -np.inf
    x[2] = np.round(x[2])
    x[3] += 100.0
    x = rounded(x, dtype)
    m = workloads.bernoulli_masks(rng, np.full(4, 0.5), 5003)
    for policy in ((1e20, 0, 1.0, 1.0), (1e300, 0, 0.5123, 1.0), (1e30, 700, 1.0, 1.0),
                   (1e30, 20, 0.77, 1.0), (1e38, 0, 1.0, 0.999)):
        check(x, None, dtype, table(policy, 4), rng.random(4))
        check(x, m, dtype, table(policy, 4), rng.random(4))
    tiny = rounded(rng.standard_normal((4, 5003)) * (1e-5 if dtype == "f16" else 1e-25), dtype)
    t = 1e13 if dtype == "f16" else 1.0
    for policy in ((t, 0, 1.0, 1.0), (t, 0, 0.5123, 1.0), (t, 30, 1.0, 1.0)):
        check(tiny, m, dtype, table(policy, 4), rng.random(4))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,vocab", [(6, 50021), (70, 128256)])
def test_masks_of_a_grammar(rows, vocab, dtype, cuda_lib):
    """A handful of valid ids, one, a long run, two runs far apart, all but a run, and a run that
    ends with the row; NaN and infinities in masked places. Kept rows and streamed ones."""
    if rows == 70:
        assert_ring(rows, vocab, dtype, True)
    rng = np.random.default_rng(150 + rows)
    x, _, u = ring_rows(rows, vocab, 0, False, dtype, 151)
    valid = np.zeros((rows, vocab), bool)
    for r in range(rows):
        a = int(rng.integers(0, vocab - 20000))
        kind = r % 6
        if kind == 0:
            valid[r, rng.integers(0, vocab, 10)] = True
        elif kind == 1:
            valid[r, a] = True
        elif kind == 2:
            valid[r, a: a + 17001] = True
        elif kind == 3:
            valid[r, :37] = valid[r, vocab - 5000:] = True
        elif kind == 4:
            valid[r] = True
            valid[r, a: a + 9000] = False
        else:
            valid[r, vocab - 3:] = True
    x = torch.where(torch.from_numpy(valid).cuda(), x, float("nan"))
    x[::2] = torch.where(x[::2].isnan(), float("inf"), x[::2])
    m = np.packbits(np.pad(valid, ((0, 0), (0, -vocab % 32))), axis=1, bitorder="little")
    m = masks_to_device(m.view(np.uint32))
    for shift in range(3):
        policies = np.stack([POLICIES[RING_POLICIES[(r // 6 + shift) % 6]] for r in range(rows)])
        r1 = ox.policy_sample(x, m, gpu(policies), u)
        probs, status = ox.policy_probs(x, m, gpu(policies))
        assert not r1.status.any() and not status.any()
        ids, numbers = host(r1.token_ids), host(u)
        for r in range(shift, rows, 1 if rows < 10 else 7):
            w = oracle_row(x[r], m[r], policies[r], numbers[r], ids[r])
            assert_probs(probs[r], w / w.sum())
