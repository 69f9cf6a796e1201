"""Performance cases of a layer whose attention is not the plain causal one: its queries and keys are normalised and
rotated on their way into the paged cache, and its scores are capped, lean on the distance or are masked.

Four kinds, each called the way a serving program calls it:

* ``append`` a step's queries and keys: RMS norm of each head, rotation by the token's position (half or interleaved
             pairs, of the whole head or its first part, frequencies scaled for long contexts), keys and values into
             their pages;
* ``rope``   the same without a cache: the rotated queries and keys come back;
* ``prompt`` attention of several new tokens a row over the paged cache: scores capped by a tanh, a bias that falls
             with the distance, a window, documents packed into a row, a prefix that is seen as a whole;
* ``single`` the same for one new token a row.

Head layouts and contexts are those of this repository's model shapes and benchmark configurations (Llama-3-8B,
Qwen2.5-7B, Qwen2.5-14B, DeepSeek-R1-Distill-Qwen-1.5B).  Row lengths come from the case alone, values from the seed.
"""
import math
import random

import torch

own = False

DEV = "cuda:0"
PAGE = 16
D = 128
EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # One decoding request: latency alone.
        {"name": "append_1", "kind": "append", "batch": 1, "hq": 12, "hkv": 2, "qlo": 1, "qhi": 1, "plo": 500, "phi": 500,
         "norm": True, "rot": 128, "inter": False, "scaling": "none", "far": 0, "lens": 1, "dtype": "bf16"},
        # A decode step of 128 ragged rows that rotates half of each head.
        {"name": "append_128", "kind": "append", "batch": 128, "hq": 40, "hkv": 8, "qlo": 1, "qhi": 1, "plo": 200, "phi": 1500,
         "norm": True, "rot": 64, "inter": False, "scaling": "linear", "far": 20000, "lens": 2, "dtype": "fp16"},
        # A long prompt's layer, positions far past the trained context.
        {"name": "append_8k", "kind": "append", "batch": 1, "hq": 32, "hkv": 8, "qlo": 8192, "qhi": 8192, "plo": 0, "phi": 0,
         "norm": True, "rot": 128, "inter": False, "scaling": "yarn", "far": 120000, "lens": 3, "dtype": "bf16"},
        # Five prompts of a model that keeps its keys elsewhere, interleaved pairs of three quarters of the head.
        {"name": "rope_5", "kind": "rope", "batch": 5, "hq": 28, "hkv": 4, "qlo": 37, "qhi": 1500, "plo": 0, "phi": 900,
         "norm": True, "rot": 96, "inter": True, "scaling": "none", "far": 0, "lens": 4, "dtype": "bf16"},
        # Three short questions, bias by distance: latency.
        {"name": "prompt_3", "kind": "prompt", "batch": 3, "hq": 12, "hkv": 2, "qlo": 5, "qhi": 40, "plo": 0, "phi": 0,
         "cap": 0.0, "slopes": True, "window": 0, "mask": "causal", "lens": 5, "dtype": "bf16"},
        # One 8192-token prompt of a layer with capped scores.
        {"name": "prompt_8k", "kind": "prompt", "batch": 1, "hq": 32, "hkv": 8, "qlo": 8192, "qhi": 8192, "plo": 0, "phi": 0,
         "cap": 50.0, "slopes": False, "window": 0, "mask": "causal", "lens": 6, "dtype": "bf16"},
        # Documents packed into two rows, each seen by its own tokens alone, bias by distance.
        {"name": "prompt_docs", "kind": "prompt", "batch": 2, "hq": 40, "hkv": 8, "qlo": 4000, "qhi": 6000, "plo": 0, "phi": 0,
         "cap": 0.0, "slopes": True, "window": 0, "mask": "docs", "lens": 7, "dtype": "fp16"},
        # A chunk of a few words at the end of a 65536-token cache whose first part is a prefix seen as a whole.
        {"name": "chunk_64k", "kind": "prompt", "batch": 1, "hq": 28, "hkv": 4, "qlo": 48, "qhi": 48, "plo": 65500, "phi": 65500,
         "cap": 30.0, "slopes": False, "window": 0, "mask": "prefix", "lens": 8, "dtype": "bf16"},
        # A mixed step of a local layer: 16 rows that bring one token or several hundred, window 1024, capped.
        {"name": "chunk_16_window", "kind": "prompt", "batch": 16, "hq": 32, "hkv": 8, "qlo": 1, "qhi": 600, "plo": 0,
         "phi": 6000, "cap": 50.0, "slopes": False, "window": 1024, "mask": "causal", "lens": 9, "dtype": "bf16"},
        # Two decoding requests of a few hundred tokens.
        {"name": "single_2", "kind": "single", "batch": 2, "hq": 12, "hkv": 2, "qlo": 1, "qhi": 1, "plo": 39, "phi": 499,
         "cap": 0.0, "slopes": True, "window": 0, "mask": "causal", "lens": 10, "dtype": "fp16"},
        # The benchmark's decode batch, 32 rows of 8192 tokens, capped.
        {"name": "single_32", "kind": "single", "batch": 32, "hq": 32, "hkv": 8, "qlo": 1, "qhi": 1, "plo": 8191, "phi": 8191,
         "cap": 50.0, "slopes": False, "window": 0, "mask": "causal", "lens": 11, "dtype": "bf16"},
        # 64 ragged rows of a local layer, window 4096, capped.
        {"name": "single_64_window", "kind": "single", "batch": 64, "hq": 40, "hkv": 8, "qlo": 1, "qhi": 1, "plo": 1000,
         "phi": 16000, "cap": 30.0, "slopes": False, "window": 4096, "mask": "causal", "lens": 12, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


# (q heads, kv heads): the model table's layouts (groups of 4, 5, 6 and 7), and groups of 1, 2, 3 and 8.
HEADS = [(32, 8), (40, 8), (12, 2), (28, 4), (32, 8), (40, 8), (12, 2), (28, 4), (4, 4), (4, 2), (12, 4), (32, 4)]
MOST_KV = 64 * 8500 * 8     # cached tokens x kv heads
MOST_DOTS = 32 * 8192 * 4096  # (query, key) pairs x q heads


def draw(rng):
    kind = rng.choice(["append", "append", "rope", "prompt", "prompt", "prompt", "single", "single"])
    hq, hkv = rng.choice(HEADS)
    case = {"kind": kind, "hq": hq, "hkv": hkv, "lens": rng.randrange(1000), "dtype": rng.choice(["bf16", "bf16", "fp16"])}
    if kind in ("append", "rope"):
        batch = _log(rng, 1, 128)
        qhi = rng.choice([1, _log(rng, 1, 8192 // batch)])
        return {**case, "batch": batch, "qlo": rng.choice([1, qhi]), "qhi": qhi, "plo": 0, "phi": rng.choice([0, 700]),
                "norm": rng.choice([True, True, False]), "rot": rng.choice([128, 128, 64, 32, 96, 2 * rng.randint(1, 64)]),
                "inter": rng.choice([False, False, True]), "scaling": rng.choice(["none", "linear", "llama31", "yarn"]),
                "far": rng.choice([0, _log(rng, 1, 1000000)])}
    batch = _log(rng, 1, 128 if kind == "single" else 32)
    most = min(65536, MOST_KV // (batch * hkv))
    phi = _log(rng, 1, most * 15 // 16)
    qhi = 1 if kind == "single" else _log(rng, 1, max(1, min(8192, most // 16, MOST_DOTS // (batch * hq * (phi + 64)))))
    if kind == "prompt" and rng.random() < 0.3:  # whole prompts
        phi, qhi = 0, _log(rng, 1, min(8192, most, int(math.sqrt(2 * MOST_DOTS / (batch * hq)))))
    mask = rng.choice(["causal", "causal", "docs", "prefix"])
    while qhi > 1 and batch * hq * qhi * (phi + (qhi if mask == "prefix" else qhi / 2)) > MOST_DOTS:
        qhi = qhi * 7 // 8
    return {**case, "batch": batch, "qlo": rng.choice([1, qhi]), "qhi": qhi, "plo": rng.choice([0, phi]), "phi": phi,
            "cap": rng.choice([0.0, 30.0, 50.0]), "slopes": rng.choice([False, False, True]),
            "window": rng.choice([0, 0, _log(rng, 1, 8192)]), "mask": mask}


# ------------------------------------------------------------------ lengths (the case alone)
def _shape(case):
    """Each row's cached tokens in front of its new ones, its new tokens, and the position of its first new one."""
    rng = random.Random(case["lens"])
    past = [rng.randint(case["plo"], case["phi"]) for _ in range(case["batch"])]
    new = [rng.randint(case["qlo"], case["qhi"]) for _ in range(case["batch"])]
    far = case.get("far", 0)
    return past, new, [p + (rng.randint(far // 2, far) if far else 0) for p in past]


def _bounds(case):
    """Each query token's position in its row, and the first key it sees and the one behind its last."""
    past, new, _ = _shape(case)
    rng = random.Random(case["lens"] + 1)
    pos, begin, end = [], [], []
    for p, n in zip(past, new):
        starts = [0]  # of the row's documents
        while case["mask"] == "docs" and starts[-1] < p + n:
            starts.append(starts[-1] + _log(rng, 1, 1500))
        prefix = rng.randint(1, p + n) if case["mask"] == "prefix" else 0
        d = 0
        for at in range(p, p + n):
            while d + 1 < len(starts) and starts[d + 1] <= at:
                d += 1
            pos.append(at)
            begin.append(starts[d])
            end.append(max(at + 1, prefix))
    return pos, begin, end


def work(case):
    past, new, _ = _shape(case)
    hq, hkv, tokens = case["hq"], case["hkv"], sum(new)
    if case["kind"] in ("append", "rope"):
        heads = hq + (2 if case["kind"] == "append" else 1) * hkv
        return {"bytes": 2 * tokens * heads * D * 2, "flops": 8 * tokens * (hq + hkv) * D}
    pos, begin, end = _bounds(case)
    if case["window"]:
        begin = [max(b, p - case["window"] + 1) for b, p in zip(begin, pos)]
    dots = sum(e - b for b, e in zip(begin, end))
    kv, t = 0, 0
    for n in new:  # the keys that some query of the row sees
        seen = 0
        for b, e in sorted(zip(begin[t:t + n], end[t:t + n])):
            if e > seen:
                kv += e - max(b, seen)
                seen = e
        t += n
    return {"bytes": kv * 2 * hkv * D * 2 + tokens * hq * (2 * D * 2 + 4), "flops": 4 * D * hq * dots}


# ------------------------------------------------------------------ inputs
def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _indptr(counts):
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return out


# What a model's configuration says of its rotation: base, factor and the trained context that it is scaled from.
THETA = 500000.0
SCALINGS = {"none": {}, "linear": {"rope_scale": 4.0},
            "llama31": {"rope_scale": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "old_context_len": 8192.0},
            "yarn": {"rope_scale": 16.0, "old_context_len": 8192.0, "scaling": "yarn"}}


def _frequencies(case):
    """Radians a position of each pair, and the factor on what is rotated (64 bits)."""
    p = SCALINGS[case["scaling"]]
    s, ctx = p.get("rope_scale", 1.0), p.get("old_context_len", 0.0)
    f = torch.tensor([THETA ** (-2.0 * j / case["rot"]) for j in range(case["rot"] // 2)], dtype=torch.float64, device=DEV)
    turns = f * (ctx / (2 * math.pi))  # over the trained context
    if case["scaling"] == "llama31":
        keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return f / s * (1 - keep) + f * keep, 1.0
    if case["scaling"] == "yarn":
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        return f / s * (1 - keep) + f * keep, 0.1 * math.log(s) + 1.0
    return f / s, 1.0


def _plan(case):
    from delta_amd import kernels as K
    return K.rotary(case["rot"], rope_theta=THETA, interleaved=case["inter"], device=DEV, **SCALINGS[case["scaling"]])


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    past, new, first = _shape(case)
    hq, hkv, kind, T = case["hq"], case["hkv"], case["kind"], sum(new)
    pages = [-(-(p + n) // PAGE) for p, n in zip(past, new)]
    order = list(range(sum(pages) + 3))  # pages of a pool in use: in no order, some of them other rows'
    random.Random(seed).shuffle(order)
    at = _indptr(pages)
    s = {"case": case, "qo_indptr": _i32(_indptr(new)), "max_qo": max(new), "kv_indptr": _i32(at),
         "kv_indices": _i32(order[:at[-1]]), "last": _i32([(p + n - 1) % PAGE + 1 for p, n in zip(past, new)]),
         "max_pages": max(pages)}
    if kind != "rope":
        s["cache"] = torch.empty(len(order), 2, PAGE, hkv, D, dtype=dtype, device=DEV).normal_(0.0, 1.0, generator=gen)
    if kind in ("append", "rope"):
        # the merged projection's output: q, k and v are views of its rows
        qkv = torch.empty(T, (hq + 2 * hkv) * D, dtype=dtype, device=DEV).normal_(0.0, 1.0, generator=gen)
        q, k, v = qkv.split([hq * D, hkv * D, hkv * D], dim=-1)
        s.update(q=q.view(T, hq, D), k=k.view(T, hkv, D), v=v.view(T, hkv, D), offsets=_i32(first), q_weight=None, k_weight=None)
        if case["norm"]:
            for name in ("q_weight", "k_weight"):
                s[name] = torch.empty(D, dtype=dtype, device=DEV).normal_(1.0, 0.2, generator=gen)
        s["frequencies"] = _frequencies(case)
        if own:
            s["rotary"] = _plan(case)
        return s
    # scores of about the size at which a cap matters, where there is one
    s["q"] = torch.empty(T, hq, D, dtype=dtype, device=DEV).normal_(0.0, 4.0 if case["cap"] else 1.5, generator=gen)
    pos, begin, end = _bounds(case)
    s["positions"] = _i32(pos)
    s["slopes"] = s["kv_begin"] = s["kv_end"] = None
    if case["slopes"]:
        s["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / hq) for h in range(hq)], dtype=torch.float32, device=DEV)
    if case["mask"] == "docs":
        s["kv_begin"] = _i32(begin)
    if case["mask"] == "prefix":
        s["kv_end"] = _i32(end)
    return s


# ------------------------------------------------------------------ plain forms
def _rows_of(s, T):
    """Each new token's row, and its place among the row's new tokens."""
    ip = s["qo_indptr"].long()
    row = torch.searchsorted(ip[1:], torch.arange(T, device=DEV), right=True)
    return row, torch.arange(T, device=DEV) - ip[row]


def _turned(x, weight, cos, sin, case):
    """Norm and rotation of [T, heads, D] in 32 bits."""
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
    r = case["rot"]
    y = x.clone()
    cos, sin = cos[:, None], sin[:, None]
    if case["inter"]:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y[..., 0:r:2], y[..., 1:r:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        y[..., :r // 2], y[..., r // 2:r] = a * cos - b * sin, b * cos + a * sin
    return y


def _append(s):
    case, T, dtype = s["case"], s["q"].shape[0], s["q"].dtype
    row, i = _rows_of(s, T)
    f, factor = s["frequencies"]
    angle = (s["offsets"].long()[row] + i).double()[:, None] * f
    cos, sin = (torch.cos(angle) * factor).float(), (torch.sin(angle) * factor).float()
    q = _turned(s["q"], s["q_weight"], cos, sin, case).to(dtype)
    k = _turned(s["k"], s["k_weight"], cos, sin, case).to(dtype)
    if case["kind"] == "rope":
        return {"q": q, "k": k}
    kv_ip, qo_ip = s["kv_indptr"].long(), s["qo_indptr"].long()
    kv_len = (kv_ip[1:] - kv_ip[:-1] - 1) * PAGE + s["last"]
    at = (kv_len - (qo_ip[1:] - qo_ip[:-1]))[row] + i
    page = s["kv_indices"].long()[kv_ip[row] + at // PAGE]
    s["cache"][page, 0, at % PAGE] = k
    s["cache"][page, 1, at % PAGE] = s["v"]
    return {"q": q, "cache": s["cache"]}


def _attend(s, rows, i0, mq):
    """Query tokens i0 .. i0 + mq of each of a run of rows over the rows' whole page lists, padded to the longest one.
    Returns o and lse, [rows, mq, hq, ..]; what lies past a row's tokens means nothing."""
    case, q, cache, kv_ip, qo_ip = s["case"], s["q"], s["cache"], s["kv_indptr"].long(), s["qo_indptr"].long()
    T, hq, _ = q.shape
    hkv = cache.shape[3]
    G = hq // hkv
    a, b = rows
    B = b - a
    npages = kv_ip[a + 1:b + 1] - kv_ip[a:b]
    mp = s["max_pages"]
    S = mp * PAGE
    key = torch.arange(S, device=DEV)
    ids = s["kv_indices"].long()[(kv_ip[a:b, None] + key[:mp]).clamp(max=s["kv_indices"].numel() - 1)]
    kv_len = (npages - 1) * PAGE + s["last"][a:b]
    kv = cache[ids]
    k = kv[:, :, 0].reshape(B, S, hkv, D).permute(0, 2, 3, 1).float().contiguous()
    v = kv[:, :, 1].reshape(B, S, hkv, D).permute(0, 2, 1, 3).float().contiguous()
    tok = (qo_ip[a:b, None] + i0 + torch.arange(mq, device=DEV)).clamp(max=T - 1)
    x = q[tok].float().view(B, mq, hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, hkv, G * mq, D).contiguous()
    z = torch.matmul(x, k).mul_(1.0 / math.sqrt(D)).view(B, hkv, G, mq, S)
    if case["cap"]:
        z.div_(case["cap"]).tanh_().mul_(case["cap"])
    pos = s["positions"].long()[tok][:, :, None]
    if s["slopes"] is not None:
        z.sub_(s["slopes"].view(1, hkv, G, 1, 1) * (pos - key).abs().float()[:, None, None])
    end = s["kv_end"].long()[tok][:, :, None] if s["kv_end"] is not None else pos + 1
    hidden = (key >= end) | (key >= kv_len[:, None, None])
    if s["kv_begin"] is not None:
        hidden |= key < s["kv_begin"].long()[tok][:, :, None]
    if case["window"]:
        hidden |= key <= pos - case["window"]
    z.masked_fill_(hidden[:, None, None], float("-inf"))
    m = z.amax(-1, keepdim=True)
    z.sub_(m).exp_()
    total = z.sum(-1, keepdim=True)
    o = torch.matmul(z.view(B, hkv, G * mq, S), v).view(B, hkv, G, mq, D) / total
    lse = (m + total.log()).squeeze(-1)
    return o.permute(0, 3, 1, 2, 4).reshape(B, mq, hq, D).to(q.dtype), lse.permute(0, 3, 1, 2).reshape(B, mq, hq)


def _attend_all(s):
    q, hkv = s["q"], s["cache"].shape[3]
    T, hq, _ = q.shape
    B, mq, S = s["qo_indptr"].numel() - 1, s["max_qo"], s["max_pages"] * PAGE
    row, tok = _rows_of(s, T)
    o, lse = torch.empty_like(q), torch.empty(T, hq, dtype=torch.float32, device=DEV)
    step = max(1, min(mq, (1 << 29) // (hq * S)))  # query tokens a time, then rows
    most = max(1, min(B, (1 << 29) // (step * hq * S), (1 << 31) // (S * hkv * D)))
    for a in range(0, B, most):
        b = min(B, a + most)
        for i0 in range(0, mq, step):
            n = min(step, mq - i0)
            po, pl = _attend(s, (a, b), i0, n)
            if most >= B and step >= mq:
                return {"o": po[row, tok], "lse": pl[row, tok]}
            here = (row >= a) & (row < b) & (tok >= i0) & (tok < i0 + n)
            o[here], lse[here] = po[row[here] - a, tok[here] - i0], pl[row[here] - a, tok[here] - i0]
    return {"o": o, "lse": lse}


def run(state):
    s = state
    case, kind = s["case"], s["case"]["kind"]
    if not own:
        return _append(s) if kind in ("append", "rope") else _attend_all(s)
    from delta_amd import kernels as K
    if kind in ("append", "rope"):
        if "rotary" not in s:
            s["rotary"] = _plan(case)
        norm = {"q_weight": s["q_weight"], "k_weight": s["k_weight"], "eps": EPS}
        if kind == "rope":
            q, k = K.qk_norm_rope(s["q"], s["k"], s["qo_indptr"], s["offsets"], s["rotary"], **norm)
            return {"q": q, "k": k}
        q = K.qk_norm_rope_append(s["q"], s["k"], s["v"], s["qo_indptr"], s["offsets"], s["cache"], s["kv_indices"],
                                  s["kv_indptr"], s["last"], s["rotary"], **norm)
        return {"q": q, "cache": s["cache"]}
    q = s["q"]
    rule = K.ScoreRule(softcap=case["cap"], slopes=s["slopes"], window=case["window"], kv_begin=s["kv_begin"],
                       kv_end=s["kv_end"])
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
    if kind == "single":
        o = K.paged_decode_rule(q, s["cache"], s["kv_indptr"], s["kv_indices"], s["last"], rule,
                                max_pages_per_row=s["max_pages"], lse=lse)
    else:
        o = K.paged_prefill_rule(q, s["cache"], s["qo_indptr"], s["kv_indptr"], s["kv_indices"], s["last"], rule,
                                 max_qo_len=s["max_qo"], lse=lse)
    return {"o": o, "lse": lse}


# ------------------------------------------------------------------ 64 bits
def _exact_append(case, s):
    """Each pair as a complex number times factor * e^(i angle)."""
    past, new, first = _shape(case)
    f, factor = _frequencies(case)
    r = case["rot"]
    pos = torch.cat([torch.arange(p, p + n, device=DEV, dtype=torch.float64) for p, n in zip(first, new)])
    turn = torch.polar(torch.full((sum(new), r // 2), factor, dtype=torch.float64, device=DEV), torch.outer(pos, f))
    out = []
    for name in ("q", "k"):
        x, w = s[name].double(), s[name + "_weight"]
        if w is not None:
            x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / D + EPS) * w.double()
        head = x[..., :r]
        pairs = head.unflatten(-1, (r // 2, 2)) if case["inter"] else head.unflatten(-1, (2, r // 2)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn[:, None])
        z = z if case["inter"] else z.transpose(-1, -2)
        out.append(torch.cat([z.flatten(-2), x[..., r:]], -1))
    if case["kind"] == "rope":
        return {"q": out[0], "k": out[1]}
    cache = s["cache"].double()
    page_at, t = s["kv_indptr"].tolist(), 0
    for b, (p, n) in enumerate(zip(past, new)):
        flat = s["kv_indices"][page_at[b]:page_at[b + 1]].long()
        row = cache[flat].transpose(0, 1).reshape(2, -1, case["hkv"], D)
        row[0, p:p + n], row[1, p:p + n] = out[1][t:t + n], s["v"][t:t + n].double()
        cache[flat] = row.reshape(2, -1, PAGE, case["hkv"], D).transpose(0, 1)
        t += n
    return {"q": out[0], "cache": cache}


def exact(case, seed):
    """From the definition in 64 bits; attention row by row, a few hundred queries a time."""
    s = prepare(case, seed)
    if case["kind"] in ("append", "rope"):
        return _exact_append(case, s)
    past, new, _ = _shape(case)
    pos, begin, end = (torch.tensor(v, dtype=torch.float64, device=DEV) for v in _bounds(case))
    hq, hkv = case["hq"], case["hkv"]
    if case["window"]:
        begin = torch.maximum(begin, pos - case["window"] + 1)
    slope = None
    if case["slopes"]:
        slope = s["slopes"].double()[:, None, None]
    page_at, os, lses, t = s["kv_indptr"].tolist(), [], [], 0
    for b, (p, n) in enumerate(zip(past, new)):
        pages = s["cache"][s["kv_indices"][page_at[b]:page_at[b + 1]].long()]
        for i in range(t, t + n, 256):
            j = min(i + 256, t + n)
            lo, hi = int(begin[i:j].min()), int(end[i:j].max())
            kv = pages[lo // PAGE:-(-hi // PAGE)].transpose(0, 1).reshape(2, -1, hkv, D)[:, lo % PAGE:][:, :hi - lo].double()
            k, v = (x.transpose(0, 1).repeat_interleave(hq // hkv, 0).contiguous() for x in kv)  # [hq, keys, D]
            z = torch.bmm(s["q"][i:j].double().transpose(0, 1).contiguous(), k.transpose(1, 2).contiguous()) / math.sqrt(D)
            if case["cap"]:
                z = case["cap"] * torch.tanh(z / case["cap"])
            at = torch.arange(lo, hi, dtype=torch.float64, device=DEV)
            if slope is not None:
                z = z - slope * (pos[i:j, None] - at).abs()
            z = torch.where((at >= begin[i:j, None]) & (at < end[i:j, None]), z, torch.full_like(z, -math.inf))
            lse = torch.logsumexp(z, -1)
            os.append(torch.bmm(torch.exp(z - lse[..., None]), v).transpose(0, 1))
            lses.append(lse.transpose(0, 1))
        t += n
    return {"o": torch.cat(os), "lse": torch.cat(lses)}
