"""Sampling under a policy of its own for each row, with the random numbers given.

Batched serving draws each row under its request's own temperature, top-k, top-p and min-p.
Three calls share that distribution:

* :func:`policy_sample` -- one id per row (beside :func:`onyx_b200.masked_sample`, which
  takes one temperature / top-p for the batch and makes its own numbers);
* :func:`policy_probs` -- the filtered, renormalised probabilities, which a draft model
  keeps for the verify;
* :func:`spec_sample` -- speculative sampling of drafted tokens (beside the greedy
  :func:`onyx_b200.spec_verify`): the tokens follow the target's distribution.

With ``top_k=0`` and ``min_p=0`` the distribution is the reference's
(onyx_cuda/src/onyx_cuda/selection.py, ``_filtered_reference_weights``, float64); the
reference has neither top-k nor min-p, and no sampled verify (its verify is greedy,
grammar_acceptance.py:166-283).

Policies are a float64 tensor on the GPU, ``[B, 4]`` (or ``[4]``: one for every row) with
the columns temperature, top_k, top_p, min_p: :func:`pack_policies` makes it from
:class:`SamplingPolicy` objects, once for as long as the batch's requests stay; its entries
may be rewritten in place between calls or graph replays. Values outside their ranges, which
the host cannot see, are reported per row as ``STATUS_BAD_POLICY``.

The three calls do not synchronise the device, and their results stay on the GPU;
:func:`pack_policies` copies from the host, which waits for the current stream.
"""

from __future__ import annotations

import math
from collections.abc import Iterable
from dataclasses import dataclass

import torch

from . import _lib
from . import masked_selection as _ms

__all__ = [
    "SamplingPolicy",
    "pack_policies",
    "policy_sample",
    "policy_probs",
    "spec_sample",
    "STATUS_BAD_POLICY",
]

STATUS_BAD_POLICY = _lib.STATUS_BAD_POLICY

_LOGIT_DTYPES = {
    torch.float32: _lib.DTYPE_F32,
    torch.float16: _lib.DTYPE_F16,
    torch.bfloat16: _lib.DTYPE_BF16,
}
_UNIFORM_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.float64: _lib.DTYPE_F64}


def _real(value: object, label: str) -> float:
    if isinstance(value, bool) or not isinstance(value, (int, float)):
        raise TypeError(f"{label} must be a real number")
    if not math.isfinite(value):
        raise ValueError(f"{label} must be finite")
    return float(value)


@dataclass(frozen=True, slots=True)
class SamplingPolicy:
    """One request's policy: ``temperature`` (0: the first maximum), ``top_k`` (0: off),
    ``top_p`` within (0, 1] (1: off), ``min_p`` within [0, 1] (0: off)."""

    temperature: float = 1.0
    top_k: int = 0
    top_p: float = 1.0
    min_p: float = 0.0

    def __post_init__(self) -> None:
        if _real(self.temperature, "temperature") < 0.0:
            raise ValueError("temperature cannot be negative")
        if isinstance(self.top_k, bool) or not isinstance(self.top_k, int):
            raise TypeError("top_k must be an integer")
        if not 0 <= self.top_k < 1 << 31:
            raise ValueError("top_k must be within [0, 2^31)")
        if not 0.0 < _real(self.top_p, "top_p") <= 1.0:
            raise ValueError("top_p must be within (0, 1]")
        if not 0.0 <= _real(self.min_p, "min_p") <= 1.0:
            raise ValueError("min_p must be within [0, 1]")

    def values(self) -> tuple[float, float, float, float]:
        """The policy as one row of the packed tensor."""
        return (float(self.temperature), float(self.top_k), float(self.top_p), float(self.min_p))


def pack_policies(policies: SamplingPolicy | Iterable[SamplingPolicy],
                  device: torch.device | str = "cuda") -> torch.Tensor:
    """float64 ``[B, 4]`` of a batch's policies, or ``[4]`` of a single one."""
    single = isinstance(policies, SamplingPolicy)
    items = (policies,) if single else tuple(policies)
    for p in items:
        if not isinstance(p, SamplingPolicy):
            raise TypeError("policies must be SamplingPolicy objects")
    rows = torch.tensor([p.values() for p in items], dtype=torch.float64).reshape(-1, 4)
    return (rows[0] if single else rows).to(device)


# the current stream's handle without a Stream object around it (2 us a call less)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(name: str, index: int, *args: object) -> None:
    """One C call on device ``index``, on its current stream; raises on an error code."""
    lib = _lib.load()
    if torch.cuda.current_device() == index:
        code = getattr(lib, name)(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            code = getattr(lib, name)(*args, _raw_stream(index))
    if code:
        _lib.check(name, code)


def _logit_code(dtype: torch.dtype) -> int:
    code = _LOGIT_DTYPES.get(dtype)
    if code is None:
        raise TypeError("policy sampling supports float32/float16/bfloat16 logits; "
                        f"got {dtype}")
    return code


def _policy_rows(policies: torch.Tensor, rows: int) -> tuple[torch.Tensor, int]:
    """The policies and their stride in doubles (0: one for every row)."""
    if not isinstance(policies, torch.Tensor):
        raise TypeError("policies must be a torch.Tensor (see pack_policies)")
    if not policies.is_cuda:
        raise ValueError("policies must be a CUDA tensor")
    if policies.dtype != torch.float64:
        raise TypeError(f"policies must be float64; got {policies.dtype}")
    shape = policies.shape
    if shape != (rows, 4) and shape != (4,):
        raise ValueError(f"policies must have shape [{rows}, 4] or [4]; got {tuple(shape)}")
    if policies.stride(-1) != 1 or (len(shape) == 2 and policies.stride(0) < 4):
        policies = policies.contiguous()
    return policies, 0 if len(shape) == 1 else policies.stride(0) if rows > 1 else 4


def _uniform_code(uniforms: torch.Tensor, shape: tuple[int, ...]) -> int:
    if not isinstance(uniforms, torch.Tensor):
        raise TypeError("uniforms must be a torch.Tensor")
    if not uniforms.is_cuda:
        raise ValueError("uniforms must be a CUDA tensor")
    code = _UNIFORM_DTYPES.get(uniforms.dtype)
    if code is None:
        raise TypeError(f"uniforms must be float32 or float64; got {uniforms.dtype}")
    if uniforms.shape != shape:
        raise ValueError(f"uniforms must have shape {list(shape)}; got {list(uniforms.shape)}")
    return code


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether a row (last dimension) of the one shares memory with a row of the other."""
    def layout(t: torch.Tensor) -> tuple[int, int, int, int]:  # first byte, step, rows, length
        size = t.element_size()
        step, count = (t.stride(0) * size, t.shape[0]) if t.dim() > 1 else (0, 1)
        return t.data_ptr(), step, count, t.shape[-1] * size

    (a0, a_step, a_rows, a_len), (b0, b_step, b_rows, b_len) = layout(a), layout(b)
    if (a.device != b.device or a0 + (a_rows - 1) * a_step + a_len <= b0
            or b0 + (b_rows - 1) * b_step + b_len <= a0):
        return False
    while a_rows and b_rows:  # the spans meet: row by row, in rising order of address
        if a0 < b0 + b_len and b0 < a0 + a_len:
            return True
        if a0 < b0:
            a0, a_rows = a0 + a_step, a_rows - 1
        else:
            b0, b_rows = b0 + b_step, b_rows - 1
    return False


def _rows_of(logits: torch.Tensor, bitmask: torch.Tensor | None):
    x = _ms._logits_2d(logits)
    code = _logit_code(x.dtype)
    rows, vocab = x.shape
    if rows > 1 and x.stride(0) < vocab:  # rows that overlap
        x = x.contiguous()
    m = None if bitmask is None else _ms._mask_2d(bitmask, rows, vocab)
    if m is not None and rows > 1 and m.stride(0) < _ms.mask_words(vocab):
        m = m.contiguous()
    return x, m, code, rows, vocab


def policy_sample(logits: torch.Tensor, bitmask: torch.Tensor | None, policies: torch.Tensor,
                  uniforms: torch.Tensor) -> _ms.MaskedArgmaxResult:
    """One draw per row of ``logits`` [B, V] (or one row [V]).

    ``bitmask`` [B, >=ceil(V/32)] packed words or None; ``policies`` float64 [B, 4] or [4];
    ``uniforms`` float32/float64 [B], each in [0, 1). ``token_ids`` is the first kept id, in
    id order, whose cumulative weight exceeds u times the kept total (-1 with a status);
    ``status`` EMPTY_MASK, ALL_NEG_INF, NAN_IN_SUPPORT or BAD_POLICY."""
    x, m, code, rows, vocab = _rows_of(logits, bitmask)
    pol, pol_stride = _policy_rows(policies, rows)
    u_code = _uniform_code(uniforms, (rows,))
    device = _ms._same_device(x, pol, uniforms, *(() if m is None else (m,)))
    if rows > 1 and uniforms.stride(0) < 1:
        uniforms = uniforms.contiguous()
    idx = torch.empty(rows, dtype=torch.int32, device=device)
    status = torch.empty(rows, dtype=torch.int32, device=device)
    if rows:
        _call("onyx_policy_sample", device.index, x.data_ptr(), code, rows, vocab,
              x.stride(0) if rows > 1 else vocab, None if m is None else m.data_ptr(),
              0 if m is None else m.stride(0), pol.data_ptr(), pol_stride, uniforms.data_ptr(),
              u_code, uniforms.stride(0) if rows > 1 else 1, idx.data_ptr(), status.data_ptr())
    return _ms.MaskedArgmaxResult(idx, status)


def policy_probs(logits: torch.Tensor, bitmask: torch.Tensor | None, policies: torch.Tensor, *,
                 out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """float32 probabilities [B, V] of every id under its row's policy, and the status.

    0 for ids that are not kept, and throughout a row with a status. ``out``: a float32
    tensor of that shape to write to, its rows at any stride of at least V (a draft step's
    ``draft_probs[:, i]``); no row of it may share memory with one of an input."""
    x, m, code, rows, vocab = _rows_of(logits, bitmask)
    pol, pol_stride = _policy_rows(policies, rows)
    if out is None:
        out = torch.empty((rows, vocab), dtype=torch.float32, device=x.device)
    else:
        if not isinstance(out, torch.Tensor):
            raise TypeError("out must be a torch.Tensor")
        if out.dtype != torch.float32 or out.shape != (rows, vocab):
            raise ValueError(f"out must be float32 [{rows}, {vocab}]; "
                             f"got {out.dtype} {list(out.shape)}")
        if (vocab > 1 and out.stride(1) != 1) or (rows > 1 and out.stride(0) < vocab):
            raise ValueError("out must have contiguous rows that do not overlap")
        if rows and any(_overlap(t, out) for t in (x, m, pol) if t is not None):
            raise ValueError("out must not share memory with an input")
    device = _ms._same_device(x, pol, out, *(() if m is None else (m,)))
    status = torch.empty(rows, dtype=torch.int32, device=device)
    if rows:
        _call("onyx_policy_probs", device.index, x.data_ptr(), code, rows, vocab,
              x.stride(0) if rows > 1 else vocab, None if m is None else m.data_ptr(),
              0 if m is None else m.stride(0), pol.data_ptr(), pol_stride, out.data_ptr(),
              out.stride(0) if rows > 1 else vocab, status.data_ptr())
    return out, status


def spec_sample(logits: torch.Tensor, bitmasks: torch.Tensor | None, drafts: torch.Tensor,
                policies: torch.Tensor, uniforms: torch.Tensor, *,
                draft_probs: torch.Tensor | None = None,
                draft_lens: torch.Tensor | None = None) -> _ms.SpecVerifyResult:
    """Speculative sampling: accept drafts while ``u q(d) < p(d)``, then draw one token.

    ``logits`` [B, G+1, V], ``bitmasks`` [B, G+1, >=ceil(V/32)] or None (row ``i`` under the
    grammar state reached by drafts ``0..i-1``, as for :func:`onyx_b200.spec_verify`),
    ``drafts`` int32 [B, G], ``policies`` float64 [B, 4] or [4], ``uniforms`` float32/float64
    [B, G+1]: number ``i`` tests draft ``i``, the last one draws the token.
    ``draft_probs`` float32 [B, G, V]: the distributions that the drafts were drawn from
    (:func:`policy_probs` of the draft model's rows); None where the drafts are certain (a
    lookup, or greedy drafting). ``draft_lens`` int32 [B]: how many of an entry's drafts
    count, 0 to G (None: all).

    ``accept_len``: drafts accepted; ``correction``: the token drawn at the first refusal
    from ``max(p - q, 0)``, or after the last acceptance from the following row (-1 with a
    status); ``status``: that of the row that ended the decision."""
    _ms._require_cuda(logits, "logits")
    code = _logit_code(logits.dtype)
    if logits.dim() != 3:
        raise ValueError(f"logits must have shape [B, G+1, V]; got {tuple(logits.shape)}")
    batch, g1, vocab = logits.shape
    gamma = g1 - 1
    if gamma < 1:
        raise ValueError("speculative sampling needs at least one draft token (G >= 1)")
    if gamma > 255:
        raise ValueError(f"at most 255 draft tokens are supported; got {gamma}")
    if vocab <= 0:
        raise ValueError("logits must have a non-empty vocabulary dimension")
    if logits.stride(2) != 1 or logits.stride(1) < vocab:
        logits = logits.contiguous()
    if bitmasks is not None:
        _ms._require_cuda(bitmasks, "bitmasks")
        words = _ms.mask_words(vocab)
        if (bitmasks.dtype not in _ms._MASK_DTYPES or bitmasks.dim() != 3
                or bitmasks.shape[:2] != (batch, g1) or bitmasks.shape[2] < words):
            raise ValueError(f"bitmasks must be int32/uint32 [{batch}, {g1}, >={words}]; "
                             f"got {tuple(bitmasks.shape)}")
        if bitmasks.stride(2) != 1 or bitmasks.stride(1) < words:
            bitmasks = bitmasks.contiguous()
    _ms._require_cuda(drafts, "drafts")
    if drafts.dtype != torch.int32 or drafts.shape != (batch, gamma):
        raise ValueError(f"drafts must be int32 [{batch}, {gamma}]")
    if (gamma > 1 and drafts.stride(1) != 1) or (batch > 1 and drafts.stride(0) < gamma):
        drafts = drafts.contiguous()
    pol, pol_stride = _policy_rows(policies, batch)
    u_code = _uniform_code(uniforms, (batch, g1))
    if uniforms.stride(1) != 1 or (batch > 1 and uniforms.stride(0) < g1):
        uniforms = uniforms.contiguous()
    q = draft_probs
    if q is not None:
        _ms._require_cuda(q, "draft_probs")
        if q.dtype != torch.float32 or q.shape != (batch, gamma, vocab):
            raise ValueError(f"draft_probs must be float32 [{batch}, {gamma}, {vocab}]; "
                             f"got {q.dtype} {list(q.shape)}")
        if (vocab > 1 and q.stride(2) != 1) or (gamma > 1 and q.stride(1) < vocab):
            q = q.contiguous()
    if draft_lens is not None:
        _ms._require_cuda(draft_lens, "draft_lens")
        if draft_lens.dtype != torch.int32 or draft_lens.shape != (batch,):
            raise ValueError(f"draft_lens must be int32 [{batch}]")
        draft_lens = draft_lens.contiguous()
    others = [t for t in (bitmasks, q, draft_lens) if t is not None]
    device = _ms._same_device(logits, drafts, pol, uniforms, *others)
    accept = torch.empty(batch, dtype=torch.int32, device=device)
    token = torch.empty(batch, dtype=torch.int32, device=device)
    status = torch.empty(batch, dtype=torch.int32, device=device)
    if batch:
        ws = torch.empty(batch * g1 * 16, dtype=torch.uint8, device=device)
        _call("onyx_spec_sample", device.index, logits.data_ptr(), code, batch, gamma, vocab,
              logits.stride(0) if batch > 1 else 0, logits.stride(1),
              None if bitmasks is None else bitmasks.data_ptr(),
              0 if bitmasks is None or batch == 1 else bitmasks.stride(0),
              0 if bitmasks is None else bitmasks.stride(1), drafts.data_ptr(),
              drafts.stride(0) if batch > 1 else gamma, None if q is None else q.data_ptr(),
              0 if q is None or batch == 1 else q.stride(0),
              vocab if q is None or gamma == 1 else q.stride(1),
              None if draft_lens is None else draft_lens.data_ptr(), pol.data_ptr(), pol_stride,
              uniforms.data_ptr(), u_code, uniforms.stride(0) if batch > 1 else g1,
              accept.data_ptr(), token.data_ptr(), status.data_ptr(), ws.data_ptr(), ws.numel())
    return _ms.SpecVerifyResult(accept, token, status)
