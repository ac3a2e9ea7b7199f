"""Measured cases of the policy sampling operators: the draw, its distribution and the
speculative verify that samples.

Every operator starts from rows of logits, a packed mask of the ids that are valid (int32
words, id t is bit t & 31 of word t >> 5; or None), and a policy for each row: temperature,
top_k, top_p and min_p, four float64 numbers a row.

* ``sample``: one id a row, drawn with a given uniform number (``policy_sample``).
* ``probs``: the filtered, renormalised probabilities of every id (``policy_probs``).
* ``spec``: speculative sampling of drafted tokens: accept while ``u q(d) < p(d)``, at the
  first refusal draw from ``max(p - q, 0)``, after the last acceptance draw from the row
  that follows (``spec_sample``).

The distribution p of a row: weights ``exp((v - max) / temperature)`` of the valid ids (a
temperature of 0 keeps the first maximum; ids at +inf share the mass alone); ids ranked by
value, lower ids first among equals; ``top_k`` keeps the first k (0: all); ``top_p`` keeps
the shortest prefix of these whose mass reaches top_p times theirs (1: all); ``min_p`` keeps
the ids whose weight is at least min_p times the largest. The draw is the first kept id, in
id order, whose cumulative weight passes u times the kept total.
"""

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
POLICIES = ("mixed", "top_p", "top_k", "min_p", "plain")


def listed():
    return [
        # one stream under a grammar at the smallest vocabulary: latency alone
        dict(name="sample_1_f32_32000", op="sample", rows=1, vocab=32000, pad=0, dtype="f32",
             mask=True, policy="top_p"),
        # one chat stream, no grammar
        dict(name="sample_1_bf16_128256", op="sample", rows=1, vocab=128256, pad=0, dtype="bf16",
             mask=False, policy="top_p"),
        # a serving batch under grammars, each request with a policy of its own
        dict(name="sample_64_bf16_masked", op="sample", rows=64, vocab=128256, pad=0,
             dtype="bf16", mask=True, policy="mixed"),
        # a large serving batch without grammars
        dict(name="sample_256_bf16", op="sample", rows=256, vocab=128256, pad=0, dtype="bf16",
             mask=False, policy="mixed"),
        # float32 logits of a padded head, seen through a view of an odd width
        dict(name="sample_64_f32_151665", op="sample", rows=64, vocab=151665, pad=271,
             dtype="f32", mask=False, policy="mixed"),
        # the largest vocabulary and batch
        dict(name="sample_1024_bf16_256000", op="sample", rows=1024, vocab=256000, pad=0,
             dtype="bf16", mask=True, policy="mixed"),
        # the draft side of one speculative stream
        dict(name="probs_1_f32_32000", op="probs", rows=1, vocab=32000, pad=0, dtype="f32",
             mask=True, policy="top_k"),
        # the draft side of a small batch
        dict(name="probs_8_bf16_masked", op="probs", rows=8, vocab=128256, pad=0, dtype="bf16",
             mask=True, policy="top_p"),
        # the draft side of a serving batch, float16
        dict(name="probs_64_f16", op="probs", rows=64, vocab=151936, pad=0, dtype="f16",
             mask=False, policy="mixed"),
        # the verify of one stream under a grammar
        dict(name="spec_1x4_bf16_masked", op="spec", rows=1, gamma=4, vocab=151936, pad=0,
             dtype="bf16", mask=True, policy="top_p", drafts="probs", ragged=False),
        # the verify of a serving batch under grammars
        dict(name="spec_32x4_bf16_masked", op="spec", rows=32, gamma=4, vocab=151936, pad=0,
             dtype="bf16", mask=True, policy="mixed", drafts="probs", ragged=False),
        # drafts looked up in the prompt, as many as were found, no draft model
        dict(name="spec_64x7_f16_ragged", op="spec", rows=64, gamma=7, vocab=128256, pad=0,
             dtype="f16", mask=False, policy="mixed", drafts="fixed", ragged=True),
    ]


def draw(rng):
    op = rng.choice(("sample", "probs", "spec"))
    vocab = int(round(math.exp(rng.uniform(math.log(1000), math.log(256000)))))
    most = {"sample": 256, "probs": 64, "spec": 32}[op]
    rows = int(round(math.exp(rng.uniform(0.0, math.log(most)))))
    case = dict(op=op, rows=rows, vocab=vocab, pad=rng.choice((0, 0, 1, 8, 271)),
                dtype=rng.choice(("f32", "f16", "bf16", "bf16")), mask=rng.random() < 0.5,
                policy=rng.choice(POLICIES))
    if op == "spec":
        case.update(gamma=rng.randint(1, 7), drafts=rng.choice(("probs", "fixed")),
                    ragged=rng.random() < 0.5)
    return case


# --------------------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------------------
def _masks(gen, rows, words):
    """Random masks of density 2^-2 to 2^-7: the AND of that many random words."""
    depth = torch.randint(2, 8, (rows, 1), generator=gen, device="cuda")
    mask = torch.full((rows, words), -1, dtype=torch.int32, device="cuda")
    for i in range(7):
        r = torch.randint(-2**31, 2**31, (rows, words), generator=gen, device="cuda",
                          dtype=torch.int32)
        mask = torch.where(depth > i, mask & r, mask)
    return mask


def _pick(gen, rows, values):
    at = torch.randint(0, len(values), (rows,), generator=gen, device="cuda")
    return torch.tensor(values, dtype=torch.float64, device="cuda")[at]


def _policies(gen, rows, kind):
    full = lambda v: torch.full((rows,), float(v), dtype=torch.float64, device="cuda")  # noqa: E731
    t, k, p, m = full(1), full(0), full(1), full(0)
    if kind == "mixed":
        t = _pick(gen, rows, (0.0, 0.6, 0.7, 0.8, 0.8, 1.0, 1.0, 1.2))
        k = _pick(gen, rows, (0, 0, 0, 20, 40, 50, 100, 1000))
        p = _pick(gen, rows, (1.0, 0.95, 0.95, 0.9, 0.9, 0.8))
        m = _pick(gen, rows, (0.0, 0.0, 0.0, 0.02, 0.05, 0.1))
    elif kind == "top_p":
        t, p = full(0.8), full(0.9)
    elif kind == "top_k":
        t, k = full(0.9), full(50)
    elif kind == "min_p":
        m = full(0.05)
    return torch.stack((t, k, p, m), dim=1).contiguous()


def _logits(gen, shape, pad, dtype):
    """N(0, 3) values in rows that are `pad` longer than what the call sees of them."""
    full = torch.randn(*shape[:-1], shape[-1] + pad, generator=gen, device="cuda")
    return full.mul_(3.0).to(DTYPES[dtype])[..., : shape[-1]]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rows, vocab, words = case["rows"], case["vocab"], (case["vocab"] + 31) // 32
    s = dict(op=case["op"], policies=_policies(gen, rows, case["policy"]))
    if case["op"] != "spec":
        s["logits"] = _logits(gen, (rows, vocab), case["pad"], case["dtype"])
        s["mask"] = _masks(gen, rows, words) if case["mask"] else None
        s["uniforms"] = torch.rand(rows, generator=gen, device="cuda")
        if case["op"] == "probs":
            s["out"] = torch.empty(rows, vocab, dtype=torch.float32, device="cuda")
        return s
    gamma = case["gamma"]
    s["logits"] = _logits(gen, (rows, gamma + 1, vocab), case["pad"], case["dtype"])
    s["mask"] = (_masks(gen, rows * (gamma + 1), words).view(rows, gamma + 1, words)
                 if case["mask"] else None)
    s["uniforms"] = torch.rand(rows, gamma + 1, generator=gen, device="cuda")
    # the draft model sees the target's logits through noise, at the request's temperature
    t = s["policies"][:, 0].clamp_min(0.1).view(rows, 1, 1)
    x = s["logits"][:, :gamma].float()
    x = x + 0.5 * torch.randn(x.shape, generator=gen, device="cuda")
    if case["mask"]:
        x = torch.where(_bits(s["mask"][:, :gamma], vocab), x, -math.inf)
    q = torch.softmax(x.double() / t, dim=-1).nan_to_num(0.0)
    u = torch.rand(rows, gamma, 1, generator=gen, device="cuda", dtype=torch.float64)
    if case["drafts"] == "fixed":  # a lookup proposes likely ids, without probabilities
        s["drafts"] = torch.argmax(q, dim=-1).int()
        s["q"] = None
    else:
        cum = q.cumsum(-1)
        at = torch.searchsorted(cum, u * cum[..., -1:], right=True)
        s["drafts"] = at.squeeze(-1).clamp_max(vocab - 1).int().contiguous()
        s["q"] = q.float().contiguous()
    s["lens"] = (torch.randint(0, gamma + 1, (rows,), generator=gen, device="cuda").int()
                 if case["ragged"] else None)
    return s


def work(case):
    rows, vocab, words = case["rows"], case["vocab"], (case["vocab"] + 31) // 32
    n = rows * (case.get("gamma", 0) + 1)
    size = n * (vocab * BYTES[case["dtype"]] + (4 * words if case["mask"] else 0)) + rows * 32
    size += n * 12  # uniforms, ids and status
    if case["op"] == "probs":
        size += 4 * n * vocab
    if case["op"] == "spec":  # drafts and their probabilities; q's rows only where p is kept
        size += rows * case["gamma"] * 8
    return {"bytes": size, "flops": 4.0 * n * vocab}


# --------------------------------------------------------------------------------------
# plain forms
# --------------------------------------------------------------------------------------
def _bits(words, vocab):
    at = torch.arange(vocab, device=words.device)
    return ((words[..., at >> 5] >> (at & 31).int()) & 1).bool()


def _kept(logits, mask, policies):
    """(weights of the kept ids in float64, 0 elsewhere; status) of each row. In 64 bits: a
    mass next to top_p, or a draw next to a boundary, decides a whole number."""
    vocab = logits.shape[-1]
    v = logits.double()
    valid = torch.ones_like(v, dtype=torch.bool) if mask is None else _bits(mask, vocab)
    empty = ~valid.any(-1)
    nan = (valid & v.isnan()).any(-1)
    v = torch.where(valid & ~v.isnan(), v, -math.inf)
    top = v.amax(-1, keepdim=True)
    low = (top.squeeze(-1) == -math.inf) & ~empty & ~nan
    status = empty.int() + 2 * low.int() + 4 * nan.int()
    t, k, p, m = (c.unsqueeze(-1) for c in policies.unbind(-1))
    first = v.argmax(-1, keepdim=True) == torch.arange(vocab, device=v.device)
    w = torch.exp((v - top) / t)
    w = torch.where(top == math.inf, (v == math.inf).double(), w)
    w = torch.where(t == 0, first.double(), w)
    order = torch.sort(v, dim=-1, descending=True, stable=True)[1]
    ranked = w.gather(-1, order)
    rank = torch.arange(vocab, device=v.device)
    keep = (k == 0) | (rank < k)
    cum = (ranked * keep).cumsum(-1)
    before = torch.nn.functional.pad(cum[..., :-1], (1, 0))
    keep &= (p == 1) | (before < p * cum[..., -1:])
    keep &= ranked >= m
    kept = torch.zeros_like(w).scatter_(-1, order, ranked * keep)
    return torch.where((status == 0).unsqueeze(-1), kept, 0.0), status


def _choose(weights, u):
    """The first id whose cumulative weight passes u times the total."""
    cum = weights.cumsum(-1)
    at = (cum <= u.double().unsqueeze(-1) * cum[..., -1:]).sum(-1)
    last = weights.shape[-1] - 1 - (weights > 0).flip(-1).int().argmax(-1)
    return torch.minimum(at, last).int()


def _plain_spec(s):
    logits, drafts, lens = s["logits"], s["drafts"].long(), s["lens"]
    rows, g1, vocab = logits.shape
    gamma = g1 - 1
    each = s["policies"].unsqueeze(1).expand(rows, g1, 4)
    kept, status = _kept(logits, s["mask"], each)
    p = kept / kept.sum(-1, keepdim=True).clamp_min(torch.finfo(torch.float64).tiny)
    u = s["uniforms"].double()
    at = torch.arange(gamma, device=p.device)
    length = torch.full((rows,), gamma, device=p.device) if lens is None else lens.long()
    p_d = p[:, :gamma].gather(-1, drafts.unsqueeze(-1)).squeeze(-1)
    if s["q"] is None:
        q = torch.zeros_like(p[:, :gamma]).scatter_(-1, drafts.unsqueeze(-1), 1.0)
    else:
        q = s["q"].double()
    q_d = q.gather(-1, drafts.unsqueeze(-1)).squeeze(-1)
    accept = (u[:, :gamma] * q_d < p_d) & (status[:, :gamma] == 0)
    accept &= at < length.unsqueeze(-1)
    taken = accept.int().cumprod(-1).sum(-1)
    row = torch.arange(rows, device=p.device)
    base = kept[row, taken]
    q_row = torch.nn.functional.pad(q, (0, 0, 0, 1))[row, taken]
    rest = (p[row, taken] - q_row).clamp_min(0.0)
    refused = (taken < length) & (rest.sum(-1) > 0)
    token = _choose(torch.where(refused.unsqueeze(-1), rest, base), u[:, gamma])
    ended = status[row, taken]
    return taken.int(), torch.where(ended == 0, token, -1), ended


def run(s):
    if own:
        import onyx_b200 as ox

        if s["op"] == "sample":
            r = ox.policy_sample(s["logits"], s["mask"], s["policies"], s["uniforms"])
            return r.token_ids, r.status
        if s["op"] == "probs":
            return ox.policy_probs(s["logits"], s["mask"], s["policies"], out=s["out"])
        r = ox.spec_sample(s["logits"], s["mask"], s["drafts"], s["policies"], s["uniforms"],
                           draft_probs=s["q"], draft_lens=s["lens"])
        return r.accept_len, r.correction, r.status
    if s["op"] == "spec":
        return _plain_spec(s)
    kept, status = _kept(s["logits"], s["mask"], s["policies"])
    if s["op"] == "sample":
        return torch.where(status == 0, _choose(kept, s["uniforms"]), -1), status
    total = kept.sum(-1, keepdim=True).clamp_min(torch.finfo(torch.float64).tiny)
    return (kept / total).float(), status


# --------------------------------------------------------------------------------------
# the definition in 64 bits, by thresholds instead of ranks
# --------------------------------------------------------------------------------------
def _exact_row(x, words, policy):
    """(kept weights, status) of one row: the cut is a value and a number of ids that hold
    it; sums run over the sorted values."""
    t, k, p, m = policy
    x = x.double()
    n = x.numel()
    if words is None:
        ids = torch.arange(n, device=x.device)
    else:
        bits = (words.long().unsqueeze(-1) >> torch.arange(32, device=x.device)) & 1
        ids = bits.flatten()[:n].nonzero().squeeze(-1)
    out = torch.zeros(n, dtype=torch.float64, device=x.device)
    v = x[ids]
    if not ids.numel():
        return out, 1
    if bool(v.isnan().any()):
        return out, 4
    top = v.max()
    if float(top) == -math.inf:
        return out, 2
    if t == 0:
        out[ids[(v == top).nonzero()[0]]] = 1.0
        return out, 0
    w = (v == top).double() if float(top) == math.inf else torch.exp((v - top) / t)
    falling, at = torch.sort(v, descending=True)
    mass = w[at]
    count = int(falling.numel()) if k == 0 else min(int(k), int(falling.numel()))
    if p < 1:
        cum = mass[:count].cumsum(0)
        count = min(count, 1 + int((cum < p * cum[-1]).sum()))
    count = min(count, int((mass[:count] >= m).sum()))
    cut = falling[count - 1]
    above, level = v > cut, v == cut
    room = count - int(above.sum())
    keep = above | (level & (level.long().cumsum(0) <= room))
    out[ids] = torch.where(keep, w, 0.0)
    return out, 0


def _exact_choice(weights, u):
    kept = weights.nonzero().squeeze(-1)
    cum = weights[kept].cumsum(0)
    at = int((cum <= u * cum[-1]).sum())
    return int(kept[min(at, kept.numel() - 1)])


def exact(case, seed):
    s = prepare(case, seed)
    policies = s["policies"].tolist()
    uniforms = s["uniforms"].double().tolist()
    rows = case["rows"]
    ids, states, probs = [], [], []
    if case["op"] != "spec":
        for r in range(rows):
            mask = None if s["mask"] is None else s["mask"][r]
            w, state = _exact_row(s["logits"][r], mask, policies[r])
            states.append(state)
            if case["op"] == "sample":
                ids.append(-1 if state else _exact_choice(w, uniforms[r]))
            else:
                probs.append(w if state else w / w.sum())
        if case["op"] == "sample":
            return torch.tensor(ids, dtype=torch.int32), torch.tensor(states, dtype=torch.int32)
        return torch.stack(probs), torch.tensor(states, dtype=torch.int32)
    drafts = s["drafts"].tolist()
    lens = [case["gamma"]] * rows if s["lens"] is None else s["lens"].tolist()
    taken = []
    for r in range(rows):
        i, token, state = 0, -1, 0
        while True:
            mask = None if s["mask"] is None else s["mask"][r, i]
            w, state = _exact_row(s["logits"][r, i], mask, policies[r])
            if state:
                break
            if i == lens[r]:
                token = _exact_choice(w, uniforms[r][-1])
                break
            p, d = w / w.sum(), drafts[r][i]
            if s["q"] is None:
                q = torch.zeros_like(p)
                q[d] = 1.0
            else:
                q = s["q"][r, i].double()
            if uniforms[r][i] * float(q[d]) < float(p[d]):
                i += 1
                continue
            rest = torch.clamp(p - q, min=0.0)
            token = _exact_choice(rest if float(rest.sum()) > 0 else w, uniforms[r][-1])
            break
        taken.append(i)
        ids.append(token)
        states.append(state)
    return tuple(torch.tensor(v, dtype=torch.int32) for v in (taken, ids, states))
