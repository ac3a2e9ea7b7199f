"""Policy sampling without a GPU: the policy object, the oracle against the reference's
fixtures and by brute force, and the refusals of the C entry points and the Python calls."""

from __future__ import annotations

import ctypes
import itertools
import math
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

import onyx_b200 as ox
from onyx_b200 import _lib
from oracle import policy as opol
from oracle import sampling as osamp
from tests.conftest import golden_values, load_golden


def test_policy_checks():
    p = ox.SamplingPolicy()
    assert p.values() == (1.0, 0.0, 1.0, 0.0)
    assert ox.SamplingPolicy(0, 50, 0.9, 0.1).values() == (0.0, 50.0, 0.9, 0.1)
    for kw, err in (
        (dict(temperature=-0.1), ValueError), (dict(temperature=math.nan), ValueError),
        (dict(temperature=math.inf), ValueError), (dict(temperature="1"), TypeError),
        (dict(temperature=True), TypeError), (dict(top_k=-1), ValueError),
        (dict(top_k=1.5), TypeError), (dict(top_k=True), TypeError),
        (dict(top_k=1 << 31), ValueError), (dict(top_p=0.0), ValueError),
        (dict(top_p=1.01), ValueError), (dict(top_p=math.nan), ValueError),
        (dict(min_p=-0.1), ValueError), (dict(min_p=1.1), ValueError),
        (dict(min_p=None), TypeError),
    ):
        with pytest.raises(err):
            ox.SamplingPolicy(**kw)


def test_pack_policies():
    rows = ox.pack_policies([ox.SamplingPolicy(0.7, 40), ox.SamplingPolicy(top_p=0.9)], "cpu")
    assert rows.dtype == torch.float64
    assert rows.tolist() == [[0.7, 40.0, 1.0, 0.0], [1.0, 0.0, 0.9, 0.0]]
    assert ox.pack_policies(ox.SamplingPolicy(min_p=0.5), "cpu").tolist() == [1.0, 0.0, 1.0, 0.5]
    assert ox.pack_policies([], "cpu").shape == (0, 4)
    with pytest.raises(TypeError):
        ox.pack_policies([(1.0, 0, 1.0, 0.0)], "cpu")


@pytest.mark.parametrize("case", load_golden("sampling_cases.json")["cases"],
                         ids=lambda c: c["name"])
def test_oracle_keeps_the_reference_set(case):
    """Temperature and top-p alone: the reference's kept ids and probabilities. The reference
    adds rounded shares, the weights here are added as they are: where the mass reaches top_p
    exactly (equal values, top_p 1/2) the reference's sum may fall an ulp short of it, and it
    keeps one id more."""
    x = golden_values(case["bits"], case["dtype"])
    if case["dtype"] == "bf16":
        x = (x.astype(np.uint32) << 16).view(np.float32)
    valid = osamp.unpack_mask(np.asarray(case["mask_words"], np.uint32), x.size)
    policy = (case["temperature"], 0, case["top_p"], 0.0)
    status, w = opol.kept_weights(x, valid, policy)
    if case["expected_status"] != "ok":
        assert status
        return
    expected = {i: float.fromhex(h) for i, h in case["expected_kept"]}
    whole = opol.kept_weights(x, valid, (case["temperature"], 0, 1.0, 0.0))[1].sum()
    if abs(w.sum() - case["top_p"] * whole) > 1e-12 * whole:
        assert set(np.flatnonzero(w > 0)) == set(expected)
    else:
        extra = set(expected) - set(np.flatnonzero(w > 0))
        assert len(extra) <= 1 and set(np.flatnonzero(w > 0)) <= set(expected)
        return
    # the reference's probabilities are shares of the whole mass, not of the kept one
    p = w / w.sum() * sum(expected.values())
    for i, e in expected.items():
        assert p[i] == pytest.approx(e, rel=1e-12)


def test_oracle_by_brute_force():
    """Five ids, every policy of a grid: the kept set from the definition, id by id."""
    rng = np.random.default_rng(0)
    for _ in range(40):
        v = rng.integers(-2, 3, 5) * 0.5
        valid = rng.random(5) < 0.8
        if not valid.any():
            continue
        for t, k, p, m in itertools.product((0.5, 2.0), (0, 1, 3), (0.3, 0.75, 1.0), (0.0, 0.4)):
            _, w = opol.kept_weights(v, valid, (t, k, p, m))
            ranked = sorted(np.flatnonzero(valid), key=lambda i: (-v[i], i))
            weight = {i: math.exp((v[i] - v[ranked[0]]) / t) for i in ranked}
            if k:
                ranked = ranked[:k]
            total, run, kept = sum(weight[i] for i in ranked), 0.0, []
            for i in ranked:
                if p < 1.0 and run >= p * total:
                    break
                run += weight[i]
                if weight[i] >= m:
                    kept.append(i)
            assert sorted(kept) == list(np.flatnonzero(w)), (v, valid, t, k, p, m)


def test_speculation_keeps_the_target_distribution():
    """Over a fine grid of numbers, the first token of speculative sampling has the target's
    distribution: q(d) of the drafts d, then acceptance or the remaining mass."""
    p_x, q_x = np.array([0.1, 1.2, 0.4, -0.3]), np.array([1.0, 0.2, 0.4, 0.0])
    policy = (1.0, 0, 1.0, 0.0)
    w = opol.kept_weights(p_x, np.ones(4, bool), policy)[1]
    q = np.exp(q_x) / np.exp(q_x).sum()
    n = 400
    got = np.zeros(4)
    for d in range(4):
        for a, b in itertools.product(range(n), range(40)):
            u = np.array([[(a + 0.5) / n, (b + 0.5) / 40]])
            taken, token, _ = opol.spec(np.stack([p_x, p_x])[None], None, np.array([[d]]),
                                        [policy], u, q[None, None])
            got[d if taken[0] else token[0]] += q[d] / (n * 40)
    # the grid places each acceptance within 1/n and each draw within 1/40 of its share
    np.testing.assert_allclose(got, w / w.sum(), atol=1 / n + 1 / 40)


def test_c_refusals(cuda_lib):
    """Every call is refused on the host before anything is launched (or is empty)."""
    f = cuda_lib.onyx_policy_sample
    one = 0x1000  # a pointer that is never read: refusals come first
    ok = [one, 2, 4, 100, 100, None, 0, one, 4, one, 0, 1, one, one, None]

    def call(fn, base, **change):
        args = list(base)
        for at, v in change.items():
            args[int(at[1:])] = v
        return fn(*args)

    bad, dtype = _lib.ERR_INVALID_ARGUMENT, _lib.ERR_UNSUPPORTED_DTYPE
    assert call(f, ok, a2=0) == _lib.OK
    for change, code in (
        (dict(a1=3), dtype), (dict(a1=9), dtype), (dict(a10=1), dtype), (dict(a10=2), dtype),
        (dict(a0=None), bad), (dict(a7=None), bad), (dict(a9=None), bad), (dict(a12=None), bad),
        (dict(a13=None), bad), (dict(a3=0), bad), (dict(a3=-5), bad), (dict(a3=1 << 31), bad),
        (dict(a2=-1), bad), (dict(a2=1 << 31), bad), (dict(a4=99), bad), (dict(a8=3), bad),
        (dict(a8=-4), bad), (dict(a11=0), bad), (dict(a5=one, a6=3), bad),
    ):
        assert call(f, ok, **change) == code, change
    f = cuda_lib.onyx_policy_probs
    ok = [one, 0, 4, 100, 100, None, 0, one, 0, one, 100, one, None]
    assert call(f, ok, a2=0) == _lib.OK
    for change, code in (
        (dict(a1=3), dtype), (dict(a9=None), bad), (dict(a11=None), bad), (dict(a10=99), bad),
        (dict(a4=1), bad), (dict(a8=2), bad), (dict(a5=one, a6=3), bad), (dict(a3=0), bad),
    ):
        assert call(f, ok, **change) == code, change
    f = cuda_lib.onyx_spec_sample
    need = cuda_lib.onyx_spec_sample_workspace_size(4, 3)
    assert need == 4 * 4 * 16
    assert cuda_lib.onyx_spec_sample_workspace_size(4, 0) == 0
    assert cuda_lib.onyx_spec_sample_workspace_size(4, 256) == 0
    assert cuda_lib.onyx_spec_sample_workspace_size(0, 3) == 0
    #     logits dt B  G  V    bs   rs   masks mb mr drafts ds  q   qb   qr   lens
    ok = [one, 2, 4, 3, 100, 400, 100, None, 0, 0, one, 3, one, 300, 100, None,
          one, 4, one, 0, 4, one, one, one, one, need, None]
    assert call(f, ok, a2=0) == _lib.OK
    for change, code in (
        (dict(a1=3), dtype), (dict(a19=2), dtype), (dict(a3=0), bad), (dict(a3=256), bad),
        (dict(a2=-1), bad), (dict(a2=1 << 23), bad), (dict(a4=0), bad), (dict(a6=99), bad),
        (dict(a7=one, a8=16, a9=3), bad), (dict(a10=None), bad), (dict(a11=2), bad),
        (dict(a14=99), bad), (dict(a16=None), bad), (dict(a17=1), bad), (dict(a18=None), bad),
        (dict(a20=3), bad), (dict(a21=None), bad), (dict(a22=None), bad), (dict(a23=None), bad),
        (dict(a24=None), _lib.ERR_WORKSPACE), (dict(a24=one + 4), _lib.ERR_WORKSPACE),
        (dict(a25=need - 1), _lib.ERR_WORKSPACE),
    ):
        assert call(f, ok, **change) == code, change


def test_calls_refuse_host_tensors():
    x, pol = torch.zeros(2, 10), ox.pack_policies(ox.SamplingPolicy(), "cpu")
    with pytest.raises(ValueError, match="CUDA"):
        ox.policy_sample(x, None, pol, torch.zeros(2))
    with pytest.raises(ValueError, match="CUDA"):
        ox.policy_probs(x, None, pol)
    with pytest.raises(ValueError, match="CUDA"):
        ox.spec_sample(x[None], None, torch.zeros(1, 1, dtype=torch.int32), pol, torch.zeros(1, 2))
    with pytest.raises(TypeError):
        ox.policy_sample([1.0], None, pol, torch.zeros(1))


# --------------------------------------------------------------------------------------
# rows that stream through a ring of slots in shared memory
# --------------------------------------------------------------------------------------
DTYPE_SIZES = {_lib.DTYPE_F32: 4, _lib.DTYPE_F16: 2, _lib.DTYPE_BF16: 2}


def layout_of(lib, rows, vocab, dtype, masked):
    out = (ctypes.c_int32 * 5)()
    assert lib.onyx_policy_layout(rows, vocab, dtype, int(masked), 148, out) == _lib.OK
    return dict(zip(("k", "warp_ids", "peaks", "keep", "smem"), out))


@pytest.fixture(scope="session")
def ring_copies(tmp_path_factory):
    """The ring's schedule, as the kernel compiles it, on the host."""
    src = Path(__file__).resolve().parent / "native" / "ring_copies.cpp"
    lib = tmp_path_factory.mktemp("ring") / "ring_copies.so"
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", str(src), "-o", str(lib)],
                   check=True)
    fn = ctypes.CDLL(str(lib)).ring_copies

    def call(id_first, n, vocab, depth):
        out = (ctypes.c_int64 * 3)()
        fn(id_first, n, vocab, 256, depth, out)
        return tuple(out)

    return call


@pytest.mark.parametrize("rows,vocab,dtype,masked", [
    (64, 128256, _lib.DTYPE_BF16, True), (256, 128256, _lib.DTYPE_BF16, False),
    (256, 32000, _lib.DTYPE_F32, False), (1, 256000, _lib.DTYPE_F16, True),
    (64, 151665, _lib.DTYPE_F32, False), (160, 151936, _lib.DTYPE_BF16, True),
    (1, 1500001, _lib.DTYPE_F32, False), (300, 33333, _lib.DTYPE_F16, True),
])
def test_ring_starts_its_own_chunks_alone(rows, vocab, dtype, masked, cuda_lib, ring_copies):
    """A warp copies each chunk of its part once, before it is read; no chunk of another
    warp's, and nothing is on its way when the slots become the lists of later passes."""
    plan = layout_of(cuda_lib, rows, vocab, dtype, masked)
    assert not plan["keep"]
    depth = 3 if dtype == _lib.DTYPE_F32 else 4
    for off in range(16 // DTYPE_SIZES[dtype]):
        end = vocab + off
        for warp in range(16 * plan["k"]):
            begin = min(warp * plan["warp_ids"], end)
            stop = min(begin + plan["warp_ids"], end)
            n = (stop - begin + 255) // 256
            assert ring_copies(begin - off, n, vocab, depth) == (0, 0, 0), (off, warp, n)


def test_layouts(cuda_lib):
    """Small batches keep their rows in shared memory; serving batches stream them."""
    bf16, f32 = _lib.DTYPE_BF16, _lib.DTYPE_F32
    assert layout_of(cuda_lib, 1, 128256, bf16, False) == dict(
        k=8, warp_ids=1024, peaks=1, keep=1, smem=layout_of(cuda_lib, 1, 128256, bf16, False)["smem"])
    assert layout_of(cuda_lib, 256, 128256, bf16, False)["k"] == 2
    assert layout_of(cuda_lib, 256, 32000, bf16, False)["k"] == 1
    assert not layout_of(cuda_lib, 1, 2_200_003, f32, False)["peaks"]
    for rows in (1, 2, 37, 64, 149, 1024):
        for vocab in (1, 255, 32000, 151936, 1 << 20, 1 << 30):
            for dtype in DTYPE_SIZES:
                for masked in (False, True):
                    p = layout_of(cuda_lib, rows, vocab, dtype, masked)
                    assert p["k"] in (1, 2, 4, 8) and p["warp_ids"] % 256 == 0
                    assert 16 * p["k"] * p["warp_ids"] >= vocab + 7
                    assert p["smem"] + 8192 <= 227 * 1024
    f = cuda_lib.onyx_policy_layout
    out, bad = (ctypes.c_int32 * 5)(), _lib.ERR_INVALID_ARGUMENT
    assert f(1, 100, 3, 0, 148, out) == _lib.ERR_UNSUPPORTED_DTYPE
    for args in ((0, 100, 0, 0, 148, out), (1, 0, 0, 0, 148, out), (1, 1 << 31, 0, 0, 148, out),
                 (1, 100, 0, 0, 0, out), (1, 100, 0, 0, 148, None)):
        assert f(*args) == bad


# --------------------------------------------------------------------------------------
# where a running sum reaches a goal
# --------------------------------------------------------------------------------------
@pytest.fixture(scope="session")
def crossings(tmp_path_factory):
    """Which of 512 threads say that the sum of their masses reaches a goal, on the host; and
    which would if each tested its own interval."""
    src = Path(__file__).resolve().parent / "native" / "warp_prefix.cpp"
    lib = tmp_path_factory.mktemp("prefix") / "warp_prefix.so"
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-ffp-contract=off",
                    str(src), "-o", str(lib)], check=True)
    fn = ctypes.CDLL(str(lib)).crossings

    def call(mass, goal):
        here, own = (ctypes.c_int32 * 512)(), (ctypes.c_int32 * 512)()
        fn(mass.ctypes.data_as(ctypes.c_void_p), ctypes.c_double(goal), here, own)
        return np.flatnonzero(here), np.flatnonzero(own)

    return call


def test_one_thread_reaches_a_goal(crossings):
    """Goals next to the ends of lanes and warps, where rounding decides: one thread writes where
    the sum reaches it, whose part ends within 512 2^-53 of there. (Of the threads' own
    intervals, some hold the same goal.)"""
    rng = np.random.default_rng(0)
    twice = 0
    for trial in range(60):
        mass = rng.random(512) ** rng.integers(1, 12)
        if trial % 3 == 1:
            mass = np.exp(-rng.random(512) * 40)
        if trial % 3 == 2:
            mass[rng.random(512) < 0.5] = 0.0
        cum = np.cumsum(mass)
        for at in (*range(20, 44), *rng.integers(0, 511, 20)):
            for steps in range(-3, 4):
                goal = cum[at] * (1.0 + steps * 2.0**-53)
                here, own = crossings(mass, goal)
                twice += own.size > 1
                assert here.size == 1, (trial, at, steps, here)
                i = int(here[0])
                slack = 512 * 2.0**-53 * cum[-1]
                assert cum[i] + slack >= goal >= (cum[i - 1] if i else 0.0) - slack
    assert twice  # else the masses test nothing
    assert crossings(mass, cum[-1] * 1.01)[0].size == 0
    assert crossings(mass, 0.0)[0].size == 0


# --------------------------------------------------------------------------------------
# outputs that share memory with an input
# --------------------------------------------------------------------------------------
def test_overlap_is_that_of_rows():
    """Rows that lie between each other's share nothing, though the spans do."""
    from onyx_b200.policy_sampling import _overlap

    both = torch.zeros(5, 2, 40)
    assert not _overlap(both[:, 0], both[:, 1])
    assert not _overlap(both[:, 1], both[:, 0])
    assert _overlap(both[:, 0], both[:, 0])
    flat = torch.zeros(5, 100)
    assert not _overlap(flat[:, :30], flat[:, 30:60])
    assert _overlap(flat[:, :31], flat[:, 30:60])
    assert _overlap(flat[:, 30:60], flat[:, :31])
    assert _overlap(flat[4:], flat) and _overlap(flat, flat[2:3])
    assert not _overlap(flat[:2], flat[2:]) and not _overlap(flat[3:], flat[:3])
    assert not _overlap(flat, torch.zeros(5, 100))
    # rows of other types and other distances
    words = flat.view(torch.int32)
    assert not _overlap(words[:, 60:64], flat[:, :60]) and _overlap(words[:, 59:64], flat[:, :60])
    line = torch.zeros(400, dtype=torch.float64)
    assert _overlap(line[:8].view(2, 4), line.view(torch.float32)[8:80].view(2, 36))
    assert not _overlap(line[:8].view(2, 4), line.view(torch.float32)[16:80].view(2, 32))
    assert not _overlap(line[20:24], line.view(torch.float32)[:320].view(4, 80)[:, :40])
    assert _overlap(line[18:24], line.view(torch.float32)[:320].view(4, 80)[:, :40])
