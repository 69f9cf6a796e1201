"""Performance cases of the operators for sequences that share a prefix.

Three kinds, each called the way a serving program calls it:

* ``decode`` one layer's decode attention of a batch whose rows share prefixes: the prefix's pages are read
             once for all its rows, every row's own pages by itself;
* ``prompt`` the same for prompts of several tokens that continue a shared prefix (causal);
* ``copy``   pages copied in every layer's cache: the page that a forked sequence goes on filling, or whole
             pages that move.

Head layouts and contexts are those of this repository's model shapes and benchmark configurations (Llama-3-8B,
Qwen2.5-7B, Qwen2.5-14B, DeepSeek-R1-Distill-Qwen-1.5B).  Row lengths come from the case alone, values from the
seed.
"""
import math
import random

import torch

own = False

DEV = "cuda:0"
PAGE = 16
D = 128
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # Two branches of a short conversation: latency alone.
        {"name": "decode_2", "kind": "decode", "batch": 2, "hq": 12, "hkv": 2, "prefixes": 1, "plo": 512, "phi": 512,
         "lone": 0, "olo": 1, "ohi": 40, "lens": 1, "dtype": "bf16"},
        # Eight questions to a long document.
        {"name": "decode_8_doc", "kind": "decode", "batch": 8, "hq": 28, "hkv": 4, "prefixes": 1, "plo": 16384,
         "phi": 16384, "lone": 0, "olo": 30, "ohi": 400, "lens": 2, "dtype": "fp16"},
        # A serving batch of 32 over one 8192-token context, answers of up to a thousand tokens.
        {"name": "decode_32", "kind": "decode", "batch": 32, "hq": 32, "hkv": 8, "prefixes": 1, "plo": 8192, "phi": 8192,
         "lone": 0, "olo": 16, "ohi": 1000, "lens": 3, "dtype": "bf16"},
        # 64 reasoning chains branched from five problems, some requests with no shared prefix beside them.
        {"name": "decode_64_five", "kind": "decode", "batch": 64, "hq": 12, "hkv": 2, "prefixes": 5, "plo": 700, "phi": 6000,
         "lone": 7, "olo": 1, "ohi": 2500, "lens": 4, "dtype": "bf16"},
        # The largest batch, with long rows of its own besides the long prefix.
        {"name": "decode_128", "kind": "decode", "batch": 128, "hq": 40, "hkv": 8, "prefixes": 1, "plo": 16384,
         "phi": 16384, "lone": 0, "olo": 64, "ohi": 2048, "lens": 5, "dtype": "bf16"},
        # Three short questions under a system prompt.
        {"name": "prompt_3", "kind": "prompt", "batch": 3, "hq": 32, "hkv": 8, "prefixes": 1, "plo": 304, "phi": 304, "lone": 0,
         "past": 0, "qlo": 1, "qhi": 17, "lens": 6, "dtype": "bf16"},
        # 32 questions of a few words to an 8192-token document.
        {"name": "prompt_32", "kind": "prompt", "batch": 32, "hq": 32, "hkv": 8, "prefixes": 1, "plo": 8192, "phi": 8192,
         "lone": 0, "past": 0, "qlo": 8, "qhi": 60, "lens": 7, "dtype": "bf16"},
        # Longer prompts over two few-shot prefixes, and one without.
        {"name": "prompt_8_two", "kind": "prompt", "batch": 8, "hq": 28, "hkv": 4, "prefixes": 2, "plo": 4000, "phi": 4500,
         "lone": 1, "past": 0, "qlo": 100, "qhi": 700, "lens": 8, "dtype": "fp16"},
        # Probing texts of five tokens appended to branched chains that already hold tokens of their own.
        {"name": "prompt_64_probe", "kind": "prompt", "batch": 64, "hq": 40, "hkv": 8, "prefixes": 1, "plo": 4096, "phi": 4096,
         "lone": 0, "past": 1500, "qlo": 5, "qhi": 5, "lens": 9, "dtype": "bf16"},
        # One sequence forked three ways: seven tokens of its last page in the caches of 28 layers.
        {"name": "copy_fork", "kind": "copy", "layers": 28, "hkv": 2, "pages": 400, "moves": 3, "sources": 1, "tlo": 7,
         "thi": 7, "dtype": "bf16"},
        # 32 sequences branched at once, last pages filled to different counts, 32 layers.
        {"name": "copy_branch", "kind": "copy", "layers": 32, "hkv": 8, "pages": 200, "moves": 64, "sources": 32, "tlo": 1,
         "thi": 16, "dtype": "bf16"},
        # Whole pages moved together: a quarter of a gigabyte a layer.
        {"name": "copy_move", "kind": "copy", "layers": 4, "hkv": 8, "pages": 9000, "moves": 4000, "sources": 4000,
         "tlo": 16, "thi": 16, "dtype": "fp16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


# (q heads, kv heads): the model table's layouts (groups of 4, 5, 6 and 7), and groups of 1, 2, 3 and 8.
HEADS = [(32, 8), (40, 8), (12, 2), (28, 4), (32, 8), (40, 8), (12, 2), (28, 4), (8, 8), (4, 2), (12, 4), (32, 4)]
MOST_READ = 128 * 18000 * 8  # rows x longest context x kv heads of the plain form's gathered copies
MOST_SCORES = 1 << 29        # its scores


def draw(rng):
    kind = rng.choice(["decode", "decode", "decode", "prompt", "prompt", "copy"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if kind == "copy":
        hkv, moves = rng.choice([2, 4, 8]), _log(rng, 1, 3000)
        layers = max(1, min(rng.choice([4, 28, 32, 48]), 100000 // (moves * hkv)))
        thi = rng.choice([16, 16, rng.randint(1, 16)])
        return {"kind": "copy", "layers": layers, "hkv": hkv, "pages": 2 * moves + _log(rng, 2, 1000), "moves": moves,
                "sources": max(1, moves // rng.choice([1, 1, 2, 7])), "tlo": rng.choice([1, thi]), "thi": thi, "dtype": dtype}
    hq, hkv = rng.choice(HEADS)
    batch = _log(rng, 1, 128 if kind == "decode" else 64)
    prefixes = min(batch, rng.choice([1, 1, 1, 2, 5]))
    lone = rng.choice([0, 0, (batch - prefixes) // 4])
    most = min(32000, MOST_READ // (batch * hkv))
    phi = _log(rng, 64, most * 3 // 4)
    case = {"kind": kind, "batch": batch, "hq": hq, "hkv": hkv, "prefixes": prefixes,
            "plo": rng.choice([phi, max(16, phi // 3)]), "phi": phi, "lone": lone}
    if kind == "decode":
        ohi = _log(rng, 1, min(4000, most // 4))
        return {**case, "olo": rng.choice([1, ohi]), "ohi": ohi, "lens": rng.randrange(1000), "dtype": dtype}
    past = rng.choice([0, 0, min(1000, most // 8)])
    qhi = _log(rng, 1, max(1, min(600, 4096 // batch, most // 8, MOST_SCORES // (batch * hq * (phi + past + 700)))))
    return {**case, "past": past, "qlo": rng.choice([1, qhi]), "qhi": qhi, "lens": rng.randrange(1000), "dtype": dtype}


# ------------------------------------------------------------------ lengths (the case alone)
def _shape(case):
    """Pages of each prefix; each row's prefix (-1: none), its own tokens and its query tokens."""
    rng = random.Random(case["lens"])
    pages = [max(1, rng.randint(case["plo"], case["phi"]) // PAGE) for _ in range(case["prefixes"])]
    row_prefix = [b % case["prefixes"] for b in range(case["batch"] - case["lone"])] + [-1] * case["lone"]
    rng.shuffle(row_prefix)
    own_len, q_len = [], []
    for p in row_prefix:
        if case["kind"] == "decode":
            q, n = 1, rng.randint(case["olo"], case["ohi"])
        else:
            q = rng.randint(case["qlo"], case["qhi"])
            n = q + rng.randint(0, case["past"])
        # a row without a prefix has a context of its own
        own_len.append(n + (rng.randint(1, case["phi"]) if p < 0 else 0))
        q_len.append(q)
    return pages, row_prefix, own_len, q_len


def _moves(case):
    rng = random.Random(case["pages"] * 31 + case["moves"])
    ids = rng.sample(range(case["pages"]), case["sources"] + case["moves"])
    src = [ids[i % case["sources"]] for i in range(case["moves"])]
    tokens = [rng.randint(case["tlo"], case["thi"]) for _ in range(case["moves"])]
    return src, ids[case["sources"]:], tokens


def work(case):
    if case["kind"] == "copy":
        token = 2 * case["hkv"] * D * 2 * case["layers"]
        src, dst, tokens = _moves(case)
        most = {}
        for s, t in zip(src, tokens):
            most[s] = max(most.get(s, 0), t)
        return {"bytes": (sum(most.values()) + sum(tokens)) * token, "flops": 0}
    pages, row_prefix, own_len, q_len = _shape(case)
    hq, hkv = case["hq"], case["hkv"]
    kv = sum(PAGE * pages[p] for p in set(row_prefix) if p >= 0) + sum(own_len)
    dots = 0
    for p, n, q in zip(row_prefix, own_len, q_len):
        before = n - q + (PAGE * pages[p] if p >= 0 else 0)
        dots += q * before + q * (q + 1) // 2
    return {"bytes": kv * 2 * hkv * D * 2 + sum(q_len) * hq * (2 * D * 2 + 4), "flops": 4 * D * hq * dots}


# ------------------------------------------------------------------ inputs
def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _indptr(counts):
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return out


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    if case["kind"] == "copy":
        src, dst, tokens = _moves(case)
        caches = torch.empty(case["layers"], case["pages"], 2, PAGE, case["hkv"], D, dtype=dtype, device=DEV)
        caches.normal_(0.0, 1.0, generator=gen)
        return {"kind": "copy", "all": caches, "caches": list(caches.unbind(0)), "src": _i32(src), "dst": _i32(dst),
                "tokens": None if case["tlo"] == PAGE else _i32(tokens)}
    pages, row_prefix, own_len, q_len = _shape(case)
    hq, hkv = case["hq"], case["hkv"]
    own_pages = [-(-n // PAGE) for n in own_len]
    total = sum(pages) + sum(own_pages)
    order = list(range(total + 3))  # pages of a pool in use: in no order, some of them other rows'
    random.Random(seed).shuffle(order)
    taken = iter(order)
    shared = [[next(taken) for _ in range(n)] for n in pages]
    rows = [(shared[p] if p >= 0 else []) + [next(taken) for _ in range(n)] for p, n in zip(row_prefix, own_pages)]
    cache = torch.empty(total + 3, 2, PAGE, hkv, D, dtype=dtype, device=DEV)
    cache.normal_(0.0, 1.0, generator=gen)
    q = torch.empty(sum(q_len), hq, D, dtype=dtype, device=DEV)
    q.normal_(0.0, 1.5, generator=gen)
    return {"kind": case["kind"], "q": q, "cache": cache, "qo_indptr": _i32(_indptr(q_len)), "max_qo": max(q_len),
            "kv_indptr": _i32(_indptr([len(r) for r in rows])), "kv_indices": _i32([p for r in rows for p in r]),
            "last": _i32([(n - 1) % PAGE + 1 for n in own_len]), "max_pages": max(len(r) for r in rows),
            "row_prefix": _i32(row_prefix), "prefix_indptr": _i32(_indptr(pages)),
            "prefix_indices": _i32([p for s in shared for p in s])}


# ------------------------------------------------------------------ plain forms
def _copy(s):
    big, src, dst = s["all"], s["src"].long(), s["dst"].long()
    if s["tokens"] is None:
        big[:, dst] = big[:, src]
        return
    keep = torch.arange(PAGE, device=big.device) < s["tokens"][:, None]
    big[:, dst] = torch.where(keep[None, :, None, :, None, None], big[:, src], big[:, dst])


def _attend(s):
    """Every row over its whole page list, gathered and padded to the longest row."""
    q, cache, kv_ip, qo_ip = s["q"], s["cache"], s["kv_indptr"].long(), s["qo_indptr"].long()
    T, hq, _ = q.shape
    hkv, B, mq, mp = cache.shape[3], kv_ip.numel() - 1, s["max_qo"], s["max_pages"]
    G, S = hq // hkv, mp * PAGE
    at = torch.arange(S, device=q.device)
    ids = s["kv_indices"].long()[(kv_ip[:-1, None] + at[:mp]).clamp(max=s["kv_indices"].numel() - 1)]
    kv_len = (kv_ip[1:] - kv_ip[:-1] - 1) * PAGE + s["last"]
    q_len = qo_ip[1:] - qo_ip[:-1]
    kv = cache[ids]
    k = kv[:, :, 0].reshape(B, S, hkv, D).permute(0, 2, 3, 1).float().contiguous()
    v = kv[:, :, 1].reshape(B, S, hkv, D).permute(0, 2, 1, 3).float().contiguous()
    i = torch.arange(mq, device=q.device)
    x = q[(qo_ip[:-1, None] + i).clamp(max=T - 1)].float().view(B, mq, hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, hkv, G * mq, D)
    z = torch.matmul(x, k).mul_(1.0 / math.sqrt(D)).view(B, hkv, G, mq, S)
    hidden = at > ((kv_len - q_len)[:, None] + i)[:, :, None]
    z.masked_fill_(hidden[:, None, None], float("-inf"))
    m = z.amax(-1, keepdim=True)
    z.sub_(m).exp_()
    total = z.sum(-1, keepdim=True)
    o = torch.matmul(z.view(B, hkv, G * mq, S), v).view(B, hkv, G, mq, D) / total
    lse = (m + total.log()).squeeze(-1)
    row = torch.searchsorted(qo_ip[1:], torch.arange(T, device=q.device), right=True)
    tok = torch.arange(T, device=q.device) - qo_ip[row]
    o = o.permute(0, 3, 1, 2, 4).reshape(B, mq, hq, D)[row, tok]
    return {"o": o.to(q.dtype), "lse": lse.permute(0, 3, 1, 2).reshape(B, mq, hq)[row, tok]}


def run(state):
    s = state
    if s["kind"] == "copy":
        if own:
            from delta_amd import kernels as K
            K.copy_pages(s["caches"], s["src"], s["dst"], tokens=s["tokens"])
        else:
            _copy(s)
        return {"caches": s["all"]}
    if not own:
        return _attend(s)
    from delta_amd import kernels as K
    q = s["q"]
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
    if s["kind"] == "decode":
        o = K.paged_decode_prefix(q, s["cache"], s["kv_indptr"], s["kv_indices"], s["last"], s["row_prefix"],
                                  s["prefix_indptr"], s["prefix_indices"], max_pages_per_row=s["max_pages"], lse=lse)
    else:
        o = K.paged_prefill_prefix(q, s["cache"], s["qo_indptr"], s["kv_indptr"], s["kv_indices"], s["last"],
                                   s["row_prefix"], s["prefix_indptr"], s["prefix_indices"], max_qo_len=s["max_qo"],
                                   lse=lse)
    return {"o": o, "lse": lse}


def exact(case, seed):
    """Row by row in 64 bits: the prefix's tokens and the row's own, one softmax over what each query may see."""
    s = prepare(case, seed)
    if case["kind"] == "copy":
        src, dst, tokens = _moves(case)
        after = s["all"].clone()
        for a, b, t in zip(src, dst, tokens):
            after[:, b, :, :t] = s["all"][:, a, :, :t]
        return {"caches": after}
    pages, row_prefix, own_len, q_len = _shape(case)
    hq, hkv = case["hq"], case["hkv"]
    cache, q = s["cache"], s["q"].double()
    shared_at, row_at = _indptr(pages), s["kv_indptr"].tolist()
    os, lses, t = [], [], 0
    for b, (p, n, ql) in enumerate(zip(row_prefix, own_len, q_len)):
        npre = pages[p] if p >= 0 else 0
        ids = s["kv_indices"][row_at[b] + npre:row_at[b + 1]]
        if npre:
            ids = torch.cat([s["prefix_indices"][shared_at[p]:shared_at[p + 1]], ids])
        tokens = cache[ids.long()].double().transpose(0, 1).reshape(2, -1, hkv, D)[:, :npre * PAGE + n]
        k, v = (x.repeat_interleave(hq // hkv, 1).transpose(0, 1).contiguous() for x in tokens)  # [hq, n, D]
        z = torch.bmm(q[t:t + ql].transpose(0, 1).contiguous(), k.transpose(1, 2).contiguous()) / math.sqrt(D)
        seen = torch.ones(ql, k.shape[1], dtype=torch.bool, device=DEV).tril(k.shape[1] - ql)
        z = torch.where(seen, z, torch.full_like(z, float("-inf")))
        lse = torch.logsumexp(z, -1)
        os.append(torch.bmm(torch.exp(z - lse[..., None]), v).transpose(0, 1))
        lses.append(lse.transpose(0, 1))
        t += ql
    return {"o": torch.cat(os), "lse": torch.cat(lses)}
