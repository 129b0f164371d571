"""The serving operators as timed cases: attention over packed prompts, attention of the newest tokens over a paged
key-value cache, writing new keys and values into the pages, copying pages.

A case is a dict of plain values.  ``op`` names the operator: ``prompt``, ``decode``, ``append`` or ``pages``.  The
sequences of a case have lengths between ``lo`` and ``hi``.  Where ``own`` is false, ``run`` computes the operators from their formulas in elementary torch operations.
"""
import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _case(name, op, **values):
    c = dict(op=op, **values)
    if name is not None:
        c["name"] = name
    return c


def _prompt(name, s, lo, hi, h, hkv, d, dtype, causal=True, prefix=0, lse=False, empty=False):
    """``prefix``: up to so many keys of each sequence come before its queries (a chunk of a longer prompt).
    ``empty``: every fifth sequence has no tokens (slots of a batch that are not in use)."""
    return _case(name, "prompt", s=s, lo=lo, hi=hi, h=h, hkv=hkv, d=d, dtype=dtype, causal=causal, prefix=prefix, lse=lse, empty=empty)


def _decode(name, s, lo, hi, h, hkv, d, dtype, page, layout, m=1, lse=False, empty=False):
    """``m``: newest tokens per sequence."""
    return _case(name, "decode", s=s, lo=lo, hi=hi, h=h, hkv=hkv, d=d, dtype=dtype, page=page, layout=layout, m=m, lse=lse, empty=empty)


def _append(name, t, hkv, d, dtype, page, layout, spread, pad):
    """``spread``: each token goes to a page of its own (a step of decoding); else tokens fill pages (prompts).
    ``pad``: so many further rows belong to no sequence."""
    return _case(name, "append", t=t, hkv=hkv, d=d, dtype=dtype, page=page, layout=layout, spread=spread, pad=pad)


def _pages(name, n, layers, hkv, d, dtype, page):
    return _case(name, "pages", n=n, layers=layers, hkv=hkv, d=d, dtype=dtype, page=page)


def listed():
    return [
        # one short prompt: the smallest call, time to first token of an idle server
        _prompt("prompt_one_short", 1, 77, 77, 32, 8, 128, "bf16"),
        # the prompts that arrived since the last step of a chat server, from one token to hundreds, grouped heads
        _prompt("prompt_chat_ragged", 48, 1, 700, 32, 8, 128, "bf16"),
        # long documents of different lengths in one batch, with the log normalizer; the largest
        _prompt("prompt_documents_lse", 4, 512, 8192, 32, 8, 128, "bf16", lse=True),
        # chunks of long prompts against all keys so far, small ungrouped heads
        _prompt("prompt_chunks_d64", 6, 129, 512, 16, 16, 64, "fp16", prefix=7000),
        # one sequence with a short history: the latency of a single user's step
        _decode("decode_one_short", 1, 300, 300, 32, 8, 128, "bf16", 16, "HND"),
        # a step of a running batch, histories of very different lengths, some slots idle
        _decode("decode_batch_ragged", 32, 200, 8192, 32, 8, 128, "bf16", 16, "HND", empty=True),
        # two very long histories, few heads, pages as the projections leave them, log normalizer (joined with other parts)
        _decode("decode_long_lse", 2, 50001, 65536, 32, 4, 128, "bf16", 64, "NHD", lse=True),
        # many short histories, ungrouped small heads
        _decode("decode_many_d64", 128, 512, 2048, 16, 16, 64, "fp16", 32, "HND"),
        # the new token of every sequence of a batch, and the rows a captured batch is padded with
        _append("append_step", 28, 8, 128, "bf16", 16, "HND", True, 4),
        # the keys and values of whole prompts
        _append("append_prompts", 16384, 8, 128, "bf16", 16, "HND", False, 37),
        # sequences that split into several continuations: the last page of each is copied
        _pages("pages_fork", 12, 1, 8, 128, "bf16", 16),
        # pages moved together in all layers' caches
        _pages("pages_compact", 700, 8, 8, 128, "bf16", 16),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "prompt", "decode", "decode", "decode", "append", "pages"])
    d, dtype, layout = rng.choice([64, 128, 128]), rng.choice(["bf16", "fp16"]), rng.choice(["HND", "NHD"])
    h, hkv = rng.choice([(32, 8), (32, 8), (16, 16), (16, 2), (8, 1), (32, 4), (24, 24), (28, 4), (40, 8), (6, 2)])
    page = rng.choice([16, 16, 32, 64, 128, 8, 1, 24])
    lse, empty = rng.random() < 0.3, rng.random() < 0.3
    if op == "prompt":
        s = _log_int(rng, 1, 64)
        hi = _log_int(rng, 16, 8192)
        lo = _log_int(rng, 1, hi)
        prefix = _log_int(rng, 16, 8192) if rng.random() < 0.25 else 0
        while s > 1 and s * h * hi * (hi + prefix) > 1 << 33:
            s //= 2
        while h * hi * (hi + prefix) > 1 << 33:
            hi, lo, prefix = hi // 2, (lo + 1) // 2, prefix // 2
        return _prompt(None, s, lo, hi, h, hkv, d, dtype, rng.random() < 0.85, prefix, lse, empty)
    if op == "decode":
        s = _log_int(rng, 1, 128)
        hi = _log_int(rng, 16, 65536)
        lo = _log_int(rng, max(1, hi // 50), hi)
        m = rng.choice([1, 1, 1, 1, 2, 4, 7])
        while s * hi * hkv * d > 2 * 65536 * 8 * 128:
            s, hi, lo = (s // 2, hi, lo) if s > 1 else (s, hi // 2, (lo + 1) // 2)
        return _decode(None, s, lo, hi, h, hkv, d, dtype, page, layout, m, lse, empty)
    if op == "append":
        t = _log_int(rng, 1, 16384)
        spread = t <= 256 and rng.random() < 0.6
        return _append(None, t, hkv, d, dtype, page, layout, spread, rng.choice([0, 0, 1, 5, 64]))
    n, layers = _log_int(rng, 1, 1024), rng.choice([1, 1, 2, 8, 16])
    page = max(page, 8)
    while n * layers * hkv * d * page > 700 * 8 * 8 * 128 * 16:
        n, layers = (n // 2, layers) if n > 1 else (n, layers // 2)
    return _pages(None, n, layers, hkv, d, dtype, page)


def _lengths(case, seed):
    """Keys per sequence, queries per sequence (host lists; queries are the newest tokens): evenly over the logarithm of the
    range, the longest one ``hi``, in an order that the seed gives."""
    c, s = case, case["s"]
    n = [int(round(c["hi"] * (c["lo"] / c["hi"]) ** (i / max(s - 1, 1)))) for i in range(s)]
    if c["empty"]:
        n[4::5] = [0] * len(n[4::5])
    q = n if c["op"] == "prompt" else [c["m"]] * s
    if c.get("prefix", 0):
        n = [x + c["prefix"] * (i * 7 % s + 1) // s for i, x in enumerate(n)]
    order = torch.randperm(s, generator=torch.Generator().manual_seed(seed)).tolist()
    return [n[i] for i in order], [q[i] for i in order]


def _cu(lengths, dev):
    return torch.tensor([0] + lengths, dtype=torch.int64).cumsum(0).to(torch.int32).to(dev)


def prepare(case, seed):
    c, dev, dt = case, torch.device("cuda:0"), DTYPES[case["dtype"]]
    g = torch.Generator(device=dev).manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=g, device=dev, dtype=torch.float32).to(dt)

    def keys(*shape):  # [..., heads, head_dim]: channels of K have offsets of their own
        return (torch.randn(shape, generator=g, device=dev) + torch.randn(shape[-2:], generator=g, device=dev)).to(dt)

    if c["op"] == "prompt":
        n, m = _lengths(c, seed)
        # q, k and v as one projection leaves them: slices of the same rows (a chunk's keys come from further back)
        qkv = randn(sum(m), c["h"] + 2 * c["hkv"], c["d"])
        q, k, v = qkv.split([c["h"], c["hkv"], c["hkv"]], dim=1)
        if c["prefix"]:
            k, v = keys(sum(n), c["hkv"], c["d"]), randn(sum(n), c["hkv"], c["d"])
        return {"case": c, "q": q, "k": k, "v": v, "cu_q": _cu(m, dev), "cu_k": _cu(n, dev), "max_q": max(m), "max_k": max(n)}
    if c["op"] == "pages":
        total = 2 * c["n"] + 3
        shape = (c["layers"], total, c["hkv"], c["page"], c["d"])
        order = torch.randperm(total, generator=g, device=dev).to(torch.int32)
        caches = [randn(*shape), randn(*shape)]
        if c["layers"] == 1:
            caches = [x[0] for x in caches]
        return {"case": c, "caches": caches, "src": order[:c["n"]].contiguous(), "dst": order[c["n"]:2 * c["n"]].contiguous()}
    page, hkv, d = c["page"], c["hkv"], c["d"]
    hnd = c["layout"] == "HND"
    if c["op"] == "append":
        need = c["t"] if c["spread"] else -(-c["t"] // page)
        total = need + need // 4 + 2
        where = torch.randperm(total, generator=g, device=dev)[:need]
        t = torch.arange(c["t"], device=dev)
        if c["spread"]:
            slots = where * page + torch.randint(0, page, (need,), generator=g, device=dev)
        else:
            slots = where[t // page] * page + t % page
        slots = torch.cat([slots, torch.full((c["pad"],), -1, device=dev)]).to(torch.int64)
        qkv = randn(c["t"] + c["pad"], 4 * hkv, d)  # k and v are slices of what the projection leaves
        k, v = qkv[:, 2 * hkv:3 * hkv], qkv[:, 3 * hkv:]
        caches = [torch.zeros((total, hkv, page, d) if hnd else (total, page, hkv, d), dtype=dt, device=dev) for _ in range(2)]
        return {"case": c, "k": k, "v": v, "caches": caches, "slots": slots}
    n, m = _lengths(c, seed)
    used = [-(-x // page) for x in n]
    total, width = sum(used) + sum(used) // 8 + 1, max(used) + 1
    order = torch.randperm(total, generator=g, device=dev).to(torch.int32)
    table = torch.zeros((c["s"], width), dtype=torch.int32, device=dev)  # entries past a sequence's pages are stale
    at = 0
    for i, x in enumerate(used):
        table[i, :x] = order[at:at + x]
        at += x
    k, v = keys(total, page, hkv, d), randn(total, page, hkv, d)
    if hnd:
        k, v = k.transpose(1, 2).contiguous(), v.transpose(1, 2).contiguous()
    q = randn(c["s"], c["h"], d) if c["m"] == 1 else randn(c["s"], c["m"], c["h"], d)
    return {"case": c, "q": q, "caches": [k, v], "table": table, "lens": torch.tensor(n, dtype=torch.int32, device=dev)}


def _attend(q, k, v, visible, scale):
    """Softmax attention from its formula in 32 bits: q [S, M, Hq, D], k, v [S, N, Hkv, D], visible [S, M, N].
    Returns o [S, M, Hq, D] in fp32, and the log normalizer [S, M, Hq]."""
    s, m, hq, d = q.shape
    hkv = k.shape[2]
    q = q.float().view(s, m, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(s, hkv, hq // hkv * m, d)
    k, v = k.float().permute(0, 2, 3, 1).contiguous(), v.float().transpose(1, 2).contiguous()
    x = torch.matmul(q, k).mul_(scale).view(s, hkv, hq // hkv, m, -1)
    x.masked_fill_(~visible[:, None, None], -math.inf)
    top = x.amax(dim=-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = x.sub_(top).exp_()
    total = p.sum(dim=-1, keepdim=True)
    o = torch.matmul(p.view(s, hkv, hq // hkv * m, -1), v).view(s, hkv, hq // hkv, m, d)
    o = torch.where(total > 0, o / total, 0.0)
    log_normalizer = (top + total.log()).squeeze(-1)
    return o.permute(0, 3, 1, 2, 4).reshape(s, m, hq, d), log_normalizer.permute(0, 3, 1, 2).reshape(s, m, hq)


def _plain_prompt(state):
    q, k, v, cu_q, cu_k, c = state["q"], state["k"], state["v"], state["cu_q"].long(), state["cu_k"].long(), state["case"]
    dev = q.device
    at_q, at_k = torch.arange(state["max_q"], device=dev), torch.arange(state["max_k"], device=dev)
    m, n = cu_q.diff(), cu_k.diff()
    rows_q = (cu_q[:-1, None] + at_q).clamp(max=q.shape[0] - 1)  # every sequence padded to the longest
    rows_k = (cu_k[:-1, None] + at_k).clamp(max=k.shape[0] - 1)
    visible = (at_k < n[:, None])[:, None, :]
    if c["causal"]:
        visible = visible & (at_k[None, None, :] <= at_q[None, :, None] + (n - m)[:, None, None])
    visible = visible.expand(-1, state["max_q"], -1)
    o, log_normalizer = _attend(q[rows_q], k[rows_k], v[rows_k], visible, c["d"] ** -0.5)
    t = torch.arange(q.shape[0], device=dev)
    seq = torch.searchsorted(cu_q[1:].contiguous(), t, right=True)
    pos = t - cu_q[seq]
    o = o[seq, pos].to(q.dtype)
    return (o, log_normalizer[seq, pos].t().contiguous()) if c["lse"] else o


def _plain_decode(state):
    c, q, table, lens = state["case"], state["q"], state["table"].long(), state["lens"]
    k, v = state["caches"]
    if c["layout"] == "HND":
        k, v = k[table].transpose(2, 3), v[table].transpose(2, 3)  # [S, pages, page, Hkv, D]
    else:
        k, v = k[table], v[table]
    s, m = q.shape[0], c["m"]
    k, v = k.reshape(s, -1, c["hkv"], c["d"]), v.reshape(s, -1, c["hkv"], c["d"])
    last = lens[:, None] - m + torch.arange(m, device=q.device)  # last key that each of the newest tokens sees
    visible = torch.arange(k.shape[1], device=q.device) <= last[:, :, None]
    o, log_normalizer = _attend(q.view(s, m, c["h"], c["d"]), k, v, visible, c["d"] ** -0.5)
    o = o.view(q.shape).to(q.dtype)
    if not c["lse"]:
        return o
    return o, log_normalizer.transpose(1, 2).reshape((s, c["h"]) if m == 1 else (s, c["h"], m)).contiguous()


def _plain_append(state):
    c, slots = state["case"], state["slots"]
    used = slots >= 0
    page, at = slots[used] // c["page"], slots[used] % c["page"]
    kc, vc = state["caches"]
    if c["layout"] == "HND":
        kc[page, :, at], vc[page, :, at] = state["k"][used], state["v"][used]
    else:
        kc[page, at], vc[page, at] = state["k"][used], state["v"][used]
    return kc, vc


def _plain_pages(state):
    kc, vc = state["caches"]
    src, dst = state["src"].long(), state["dst"].long()
    if kc.dim() == 5:
        kc[:, dst], vc[:, dst] = kc[:, src], vc[:, src]
    else:
        kc[dst], vc[dst] = kc[src], vc[src]
    return kc, vc


def run(state):
    c = state["case"]
    if not own:
        return {"prompt": _plain_prompt, "decode": _plain_decode, "append": _plain_append, "pages": _plain_pages}[c["op"]](state)
    import flag_attn

    if c["op"] == "prompt":
        return flag_attn.flash_attention_varlen(state["q"], state["k"], state["v"], state["cu_q"], state["cu_k"], c["causal"],
                                                return_log_normalizer=c["lse"])
    if c["op"] == "decode":
        return flag_attn.paged_attention(state["q"], *state["caches"], state["table"], state["lens"], tensor_layout=c["layout"],
                                         return_log_normalizer=c["lse"])
    if c["op"] == "append":
        flag_attn.append_to_cache(state["k"], state["v"], *state["caches"], state["slots"], tensor_layout=c["layout"])
    else:
        flag_attn.copy_pages(*state["caches"], state["src"], state["dst"])
    return tuple(state["caches"])


def _pairs(n, m, causal):
    """(query, key) pairs that m queries behind n - m keys look at."""
    if not causal:
        return m * n
    m = min(m, n)  # (further queries see no key)
    return m * n - m * (m - 1) // 2


def work(case):
    """Multiply-adds of Q.K^T and P.V over the visible pairs, counted twice each; inputs read once, outputs written once."""
    c = case
    if c["op"] == "pages":
        return {"bytes": 2 * 2 * 2 * c["n"] * c["layers"] * c["hkv"] * c["page"] * c["d"] + 8 * c["n"], "flops": 0}
    if c["op"] == "append":
        return {"bytes": 2 * 2 * 2 * c["t"] * c["hkv"] * c["d"] + 8 * (c["t"] + c["pad"]), "flops": 0}
    n, m = _lengths(case, 0)
    h, hkv, d, rows = c["h"], c["hkv"], c["d"], sum(m)
    pairs = sum(_pairs(x, y, c["op"] == "decode" or c["causal"]) for x, y in zip(n, m))
    lists = 4 * (len(n) + sum(-(-x // c["page"]) for x in n)) if c["op"] == "decode" else 8 * (len(n) + 1)
    return {"bytes": 4 * rows * h * d + 4 * sum(n) * hkv * d + lists + (4 * rows * h if c["lse"] else 0), "flops": 4 * h * d * pairs}


def _exact_head(q, k, v, offset, causal):
    """One head of one sequence in 64 bits: q [M, D] against k, v [N, D]; query i sees keys up to i + offset (all: not causal)."""
    m, n = q.shape[0], k.shape[0]
    o = torch.zeros((m, q.shape[1]), dtype=torch.float64, device=q.device)
    log_normalizer = torch.full((m,), -math.inf, dtype=torch.float64, device=q.device)
    for r in range(0, m, 2048):
        e = min(r + 2048, m)
        hi = min(n, e + offset) if causal else n  # keys that any of these rows sees
        if hi <= 0:
            continue
        x = (q[r:e].double() @ k[:hi].double().t()) / math.sqrt(q.shape[1])
        if causal:
            i = torch.arange(r, e, device=q.device)[:, None] + offset
            x = torch.where(torch.arange(hi, device=q.device)[None, :] <= i, x, -math.inf)
        norm = torch.logsumexp(x, dim=1)
        sees = norm > -math.inf
        w = torch.exp(x - torch.where(sees, norm, 0.0)[:, None])
        o[r:e] = w @ v[:hi].double()
        log_normalizer[r:e] = norm
    return o, log_normalizer


def exact(case, seed):
    c = case
    state = prepare(case, seed)
    if c["op"] == "append":  # (nothing is computed: row by row what was written where)
        slots = state["slots"].tolist()
        rows = [(t, x // c["page"], x % c["page"]) for t, x in enumerate(slots) if x >= 0]
        for src, cache in zip((state["k"], state["v"]), state["caches"]):
            by_token = cache.transpose(1, 2) if c["layout"] == "HND" else cache  # [pages, page, Hkv, D]
            flat = torch.zeros_like(by_token, memory_format=torch.contiguous_format).view(-1, c["hkv"], c["d"])
            flat.index_copy_(0, torch.tensor([p * c["page"] + i for _, p, i in rows], device=flat.device),
                             src.index_select(0, torch.tensor([t for t, _, _ in rows], device=flat.device)))
            by_token.copy_(flat.view(by_token.shape))
        return tuple(state["caches"])
    if c["op"] == "pages":
        for cache in state["caches"]:
            pages = cache.unsqueeze(0) if cache.dim() == 4 else cache
            before = pages.clone()
            for a, b in zip(state["src"].tolist(), state["dst"].tolist()):
                pages[:, b].copy_(before[:, a])
        return tuple(state["caches"])
    n, m = _lengths(case, seed)
    q, group = state["q"], c["h"] // c["hkv"]
    if c["op"] == "prompt":
        o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
        norm = torch.zeros((c["h"], q.shape[0]), dtype=torch.float64, device=q.device)
        at_q = at_k = 0
        for nn, mm in zip(n, m):
            for h in range(c["h"] if mm else 0):
                k, v = state["k"][at_k:at_k + nn, h // group], state["v"][at_k:at_k + nn, h // group]
                o[at_q:at_q + mm, h], norm[h, at_q:at_q + mm] = _exact_head(q[at_q:at_q + mm, h], k, v, nn - mm, c["causal"])
            at_q, at_k = at_q + mm, at_k + nn
        return (o, norm) if c["lse"] else o
    q = q.view(c["s"], c["m"], c["h"], c["d"])
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    norm = torch.full((c["s"], c["h"], c["m"]), -math.inf, dtype=torch.float64, device=q.device)
    kc, vc = (x if c["layout"] == "NHD" else x.transpose(1, 2) for x in state["caches"])
    for i, nn in enumerate(n):
        pages = state["table"][i, :-(-nn // c["page"])].long()
        k, v = (x[pages].reshape(-1, c["hkv"], c["d"])[:nn] for x in (kc, vc))
        for h in range(c["h"]):
            o[i, :, h], norm[i, h] = _exact_head(q[i, :, h], k[:, h // group], v[:, h // group], nn - c["m"], True)
    o = o.view(state["q"].shape)
    return (o, norm if c["m"] > 1 else norm[:, :, 0]) if c["lse"] else o
