"""Measured cases of the shared-prefix MLA and of the token sampler.

Both operators belong to drawing several continuations of one committed
history: every continuation attends to the same history rows (read and scored
once for all of them) and to a short tail of its own, and the next token of each
is drawn from its row of the LM head's logits.

``run`` computes either the plain form (elementary FP32 torch operations) or,
with ``own`` set, calls the framework's operators.
"""

import math

import torch

own = False

D, DV = 576, 512          # absorbed MLA record: 512 latent dims (the values) + 64 RoPE dims
SCALE = 0.1352            # softmax scale of the V3.2 configuration
FIXED = float(2 ** 36)    # sampling weights are whole multiples of 2^-36 of the top token's weight


# ------------------------------------------------------------------- cases
def _prefix(name, B, T, H, P, S, lens="ragged", lse=False):
    return {"name": name, "op": "prefix", "B": B, "T": T, "H": H, "P": P, "S": S, "lens": lens, "lse": lse}


def _sample(name, R, V, mode, dtype="fp32"):
    return {"name": name, "op": "sample", "R": R, "V": V, "mode": mode, "dtype": dtype}


def listed():
    return [
        # Two continuations of a very short history, first step: latency only.
        _prefix("prefix_b2_p64_first_step", 2, 1, 128, 64, 1, "full"),
        # Eight continuations at the indexer's selection width (all history rows are attended).
        _prefix("prefix_b8_p2032_s16", 8, 1, 128, 2032, 16, "full"),
        # Odd history, tails of different lengths (some empty): candidates at different stages; LSE kept for a merge.
        _prefix("prefix_b5_p1999_ragged", 5, 1, 128, 1999, 33, "ragged", True),
        # Few continuations of the benchmark's 64K history: the history has to be split over the SMs.
        _prefix("prefix_b4_p65536_s8", 4, 1, 128, 65536, 8, "full"),
        # Many continuations of a long history: the tensor cores bound it.  The largest case.
        _prefix("prefix_b64_p16384_s64", 64, 1, 128, 16384, 64, "ragged"),
        # A tensor-parallel share of the heads (16): several continuations fill one row tile.
        _prefix("prefix_h16_b24_p4096", 24, 1, 16, 4096, 40, "ragged"),
        # Candidate lists of four tokens each, scored in one call (causal inside the tail).
        _prefix("prefix_b16_t4_p8191", 16, 4, 128, 8191, 12, "full"),
        # Next token of one continuation over the V3.2 vocabulary, top-k and top-p.
        _sample("sample_r1_v129280_topk_topp", 1, 129280, "topk_topp"),
        # Sixteen requests, each with its own temperature and filters.
        _sample("sample_r16_v129280_mixed", 16, 129280, "mixed"),
        # A large batch, nucleus only (flat rows keep tens of thousands of tokens).
        _sample("sample_r256_v129280_topp", 256, 129280, "topp"),
        # An odd vocabulary in BF16 logits, temperature alone.
        _sample("sample_r64_v32003_bf16_plain", 64, 32003, "plain", "bf16"),
        # The tiny configuration's vocabulary: the smallest call, min-p.
        _sample("sample_r3_v1024_minp", 3, 1024, "minp"),
    ]


_MAX_PREFIX_ROWS_KEYS = 64 * 128 * (16384 + 64)


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    if rng.random() < 0.55:
        H = rng.choice([16, 20, 64, 128, 128, 128])
        T = rng.choice([1, 1, 1, 2, 3, 4])
        B = _log_int(rng, 1, 64)
        S = max(T, _log_int(rng, 1, 128))
        P = _log_int(rng, 1, 65536)
        P = max(1, min(P, _MAX_PREFIX_ROWS_KEYS // (B * T * H) - S))
        return {"op": "prefix", "B": B, "T": T, "H": H, "P": P, "S": S, "lens": rng.choice(["full", "ragged"]),
                "lse": rng.random() < 0.5}
    return {"op": "sample", "R": _log_int(rng, 1, 256), "V": _log_int(rng, 33, 129280),
            "mode": rng.choice(["topk_topp", "mixed", "topp", "plain", "minp"]), "dtype": rng.choice(["fp32", "bf16"])}


def _lens(case):
    """Visible tail tokens of each continuation (the last query token's view)."""
    B, S = case["B"], case["S"]
    if case["lens"] == "full":
        return [S] * B
    return [(b * 37 + 11) % (S + 1) for b in range(B)]


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    if case["op"] == "prefix":
        B, T, H, P, S = (case[k] for k in "BTHPS")
        q = (randn(B, T, H, D) * 0.5).bfloat16()
        if T == 1:
            q = q[:, 0].contiguous()
        prefix = randn(P, D).bfloat16()
        tail = randn(B, S + 3, D).bfloat16()[:, :S]  # a view of a tail cache with room for more steps
        lens = torch.tensor(_lens(case), dtype=torch.int32, device="cuda")
        return {"case": case, "q": q, "prefix": prefix, "tail": tail, "lens": lens}
    R, V, mode = case["R"], case["V"], case["mode"]
    # Language-model-like rows: a Gaussian bulk with an exponential upper tail; odd rows are flatter.
    bulk = randn(R, V) * 2.0
    bulk -= torch.rand((R, V), generator=gen, device="cuda").clamp_min_(1e-12).log_() * 1.1
    bulk *= (1.0 - 0.5 * (torch.arange(R, device="cuda") % 2))[:, None]
    logits = bulk.bfloat16() if case["dtype"] == "bf16" else bulk
    u = torch.rand(R, generator=gen, device="cuda")
    params = {"temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0}
    if mode == "topk_topp":
        params.update(temperature=0.7, top_k=50, top_p=0.95)
    elif mode == "topp":
        params.update(temperature=0.8, top_p=0.9)
    elif mode == "plain":
        params.update(temperature=1.3)
    elif mode == "minp":
        params.update(min_p=0.05)
    else:  # one setting per request
        i = torch.arange(R, device="cuda")
        params = {"temperature": torch.tensor([0.0, 0.6, 1.0, 1.5], device="cuda")[i % 4],
                  "top_k": torch.tensor([0, 20, 1000], dtype=torch.int32, device="cuda")[i % 3],
                  "top_p": torch.tensor([1.0, 0.9, 0.99, 0.5, 0.95], device="cuda")[i % 5],
                  "min_p": torch.tensor([0.0, 0.02], device="cuda")[i % 2]}
    return {"case": case, "logits": logits, "u": u, "params": params}


# -------------------------------------------------------------- plain forms
def _visible(q, tail, lens):
    """[B, T, S] truth values: tail token s is visible to query token t of continuation b."""
    B, T, S = q.shape[0], q.shape[1], tail.shape[1]
    t = torch.arange(T, device=q.device)
    s = torch.arange(S, device=q.device)
    return s[None, None, :] < (lens[:, None] - (T - 1) + t[None, :])[..., None]


def _prefix_plain(q, prefix, tail, lens, scale):
    """softmax over [history rows, own visible tail rows] of scale * q . k, times their first 512 dims."""
    shape = q.shape
    if q.dim() == 3:
        q = q[:, None]
    vis = _visible(q, tail, lens)
    q = q.float()
    prefix = prefix.float()
    # Rows no query token of the continuation sees may hold anything: they count as zeros.
    tail = torch.where(vis.any(1)[..., None], tail.float(), torch.zeros((), device=q.device))
    s_p = torch.matmul(q, prefix.t()) * scale                                       # [B, T, H, P]
    s_t = torch.matmul(q, tail[:, None].transpose(2, 3)) * scale                    # [B, T, H, S]
    s_t = torch.where(vis[:, :, None, :], s_t, torch.full((), -math.inf, device=q.device))
    scores = torch.cat((s_p, s_t), -1)
    del s_p, s_t
    top = scores.amax(-1, keepdim=True)
    base = torch.where(top > -math.inf, top, torch.zeros((), device=q.device))
    w = torch.exp(scores - base)
    del scores
    total = w.sum(-1, keepdim=True)
    P = prefix.shape[0]
    out = torch.matmul(w[..., :P], prefix[:, :DV]) + torch.matmul(w[..., P:], tail[:, None, :, :DV])
    out = torch.where(total > 0, out / total, torch.zeros((), device=q.device))
    lse = (base + torch.log(total))[..., 0]
    return out.reshape(*shape[:-1], DV), lse.reshape(shape[:-1])


def _sample_plain(logits, u, temperature, top_k, top_p, min_p):
    R, V = logits.shape
    dev = logits.device

    def column(v, dtype):
        return torch.as_tensor(v, device=dev).to(dtype).expand(R)[:, None]

    T, k = column(temperature, torch.float32), column(top_k, torch.int64)
    p, mp = column(top_p, torch.float32), column(min_p, torch.float32)
    x = logits.float()
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    top, best = x.max(-1, keepdim=True)
    best = (x == top).to(torch.int8).argmax(-1, keepdim=True)
    zero = torch.zeros((), device=dev)
    d = torch.where(x == top, zero, (x - top) / torch.where(T > 0, T, torch.ones_like(T)))
    w = torch.where(x == -math.inf, zero, torch.exp(d))
    W = (w * FIXED).to(torch.int64)
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    Ws = W.gather(1, order)
    pos = torch.arange(V, device=dev)[None, :]
    keep = (pos < k) | (k <= 0)
    total_k = (Ws * keep).sum(-1, keepdim=True)
    before = Ws.cumsum(-1) - Ws
    keep &= (before.double() < p.double() * total_k.double()) | ~(p < 1)
    keep &= ~(w.gather(1, order) < mp)
    keep[:, 0] = True
    Wk = W * torch.zeros_like(keep).scatter_(1, order, keep)
    cum = Wk.cumsum(-1)
    total = cum[:, -1:]
    r = torch.minimum((u.double()[:, None] * total.double()).floor().to(torch.int64), total - 1)
    token = torch.searchsorted(cum, r, right=True).clamp_max(V - 1)
    logp = d.gather(1, token).double() - torch.log(total.double() / FIXED)
    greedy = ~(T > 0)
    token = torch.where(greedy, best, token)
    logp = torch.where(greedy, torch.zeros_like(logp), logp)
    empty = top == -math.inf
    token = torch.where(empty, torch.full_like(token, -1), token)
    logp = torch.where(empty, torch.full_like(logp, -math.inf), logp)
    return token[:, 0], logp[:, 0].float()


def run(state):
    case = state["case"]
    if case["op"] == "prefix":
        q, prefix, tail, lens = state["q"], state["prefix"], state["tail"], state["lens"]
        if own:
            from cxldsagr_b200 import ops

            return ops.shared_prefix_mla(q, prefix, tail, lens, SCALE, return_lse=case["lse"])
        out, lse = _prefix_plain(q, prefix, tail, lens, SCALE)
        out = out.bfloat16()
        return (out, lse) if case["lse"] else out
    if own:
        from cxldsagr_b200 import ops

        return ops.sample_tokens(state["logits"], state["u"], **state["params"])
    return _sample_plain(state["logits"], state["u"], **state["params"])


# --------------------------------------------------------------- definition
def exact(case, seed):
    """The outputs from the operators' definitions in 64 bits, one continuation (row) at a time."""
    st = prepare(case, seed)
    if case["op"] == "prefix":
        q = st["q"] if st["q"].dim() == 4 else st["q"][:, None]
        B, T, H, _ = q.shape
        keys = st["prefix"].double()
        out = torch.empty((B, T, H, DV), dtype=torch.float64, device="cuda")
        lse = torch.empty((B, T, H), dtype=torch.float64, device="cuda")
        for b, n in enumerate(_lens(case)):
            for t in range(T):
                seen = max(0, n - (T - 1 - t))
                rows = torch.cat((keys, st["tail"][b, :seen].double()))
                a = SCALE * (q[b, t].double() @ rows.T)
                lse[b, t] = torch.logsumexp(a, -1)
                out[b, t] = torch.softmax(a, -1) @ rows[:, :DV]
        shape = st["q"].shape[:-1]
        out, lse = out.reshape(*shape, DV), lse.reshape(shape)
        return (out, lse) if case["lse"] else out
    R, V = case["R"], case["V"]
    tokens = torch.empty(R, dtype=torch.int64, device="cuda")
    logps = torch.empty(R, dtype=torch.float64, device="cuda")

    def of(name, r):
        v = st["params"][name]
        return float(v[r]) if torch.is_tensor(v) else float(torch.tensor(v, dtype=torch.float32))

    for r in range(R):
        x = st["logits"][r].double()
        T, k, p, mp = of("temperature", r), int(of("top_k", r)), of("top_p", r), of("min_p", r)
        ranked, ids = torch.sort(x, descending=True, stable=True)
        if T == 0:
            tokens[r], logps[r] = ids[0], 0.0
            continue
        w = torch.exp((ranked - ranked[0]) / T)
        mass = torch.floor(w * FIXED)
        n = V if k <= 0 else min(k, V)
        if p < 1:
            reached = mass[:n].cumsum(0) >= p * mass[:n].sum()
            n = min(n, int(torch.nonzero(reached)[0]) + 1)
        n = max(1, min(n, int((w >= mp).sum())))
        kept, by_id = torch.sort(ids[:n])
        cum = mass[:n][by_id].cumsum(0)
        target = min(math.floor(float(st["u"][r]) * float(cum[-1])), float(cum[-1]) - 1)
        j = int(torch.nonzero(cum > target)[0])
        tokens[r] = kept[j]
        logps[r] = (ranked[:n][by_id][j] - ranked[0]) / T - torch.log(cum[-1] / FIXED)
    return tokens, logps


# --------------------------------------------------------------------- work
def work(case):
    """Each input read once, each output written once; products and sums of the visible entries."""
    if case["op"] == "prefix":
        B, T, H, P = (case[k] for k in "BTHP")
        lens = _lens(case)
        pairs = sum(H * (P + max(0, n - (T - 1 - t))) for n in lens for t in range(T))
        rows = B * T * H
        nbytes = rows * (D + DV) * 2 + (P + sum(lens)) * D * 2 + B * 4 + (rows * 4 if case["lse"] else 0)
        return {"bytes": nbytes, "flops": 2 * pairs * (D + DV)}
    R, V = case["R"], case["V"]
    size = 2 if case["dtype"] == "bf16" else 4
    # Difference, quotient, exponential and running sum per logit.
    return {"bytes": R * V * size + R * 16 + (R * 16 if case["mode"] == "mixed" else 0), "flops": 4 * R * V}
