"""The paged-cache operators' cases: storing quantised K/V rows, reading them back, attention of
decode tokens, verify passes and prefill chunks over the pages, and the verification of drafts.

`own` False computes each operator in elementary torch operations in 32 bits; True calls the
library's operators. Lengths of a ragged case follow from its `lens` alone, so that its work is
known; the values follow from the seed.
"""
from __future__ import annotations

import importlib
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
CODE_BYTES = {"bf16": 2, "int8": 1, "e4m3": 1}
PAGE_DTYPES = {"bf16": torch.bfloat16, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "e4m3": 448.0}

_pages = None


def _paged():
    global _pages
    if _pages is None:
        import __graft_entry__ as entry
        entry.load_package()
        _pages = importlib.import_module(entry.PKG_NAME + ".paged")
    return _pages


# ------------------------------------------------------------------------------------ cases

def listed():
    return [
        # One decode step's 64 columns into a sliding layer's cache (1 KV head of 256), and the
        # same rows read back.
        {"name": "store_step", "op": "store", "tokens": 64, "kv_heads": 1, "head_dim": 256,
         "page": 64, "format": "int8", "dtype": "f32", "pages": 640},
        # Several prefill chunks stored at once in a cache of 8 KV heads, bf16 rows to e4m3.
        {"name": "store_chunks", "op": "store", "tokens": 16389, "kv_heads": 8, "head_dim": 128,
         "page": 16, "format": "e4m3", "dtype": "bf16", "pages": 2049},
        # A short shared prefix handed to a host-side check.
        {"name": "read_prefix", "op": "read", "tokens": 129, "kv_heads": 1, "head_dim": 512,
         "page": 32, "format": "int8", "dtype": "f32", "pages": 512},
        # A long context moved out of the pages (offload, another engine's layout).
        {"name": "read_context", "op": "read", "tokens": 40001, "kv_heads": 8, "head_dim": 128,
         "page": 64, "format": "e4m3", "dtype": "bf16", "pages": 1024},
        # The smallest attention call: one sequence's decode token in a sliding layer.
        {"name": "decode_one", "op": "attention", "batch": 1, "q_lo": 1, "q_hi": 1, "kv_lo": 300,
         "kv_hi": 300, "heads": 8, "kv_heads": 1, "head_dim": 256, "window": 512, "page": 64,
         "format": "int8", "dtype": "bf16", "lens": 1},
        # Batched decode, 64 sequences of ragged context 128..4096 in a global layer.
        {"name": "decode_ragged", "op": "attention", "batch": 64, "q_lo": 1, "q_hi": 1,
         "kv_lo": 128, "kv_hi": 4096, "heads": 8, "kv_heads": 1, "head_dim": 512, "window": 0,
         "page": 64, "format": "int8", "dtype": "bf16", "lens": 2},
        # Few long contexts, grouped heads, f32 activations.
        {"name": "decode_long_f32", "op": "attention", "batch": 4, "q_lo": 1, "q_hi": 1,
         "kv_lo": 40000, "kv_hi": 65537, "heads": 32, "kv_heads": 8, "head_dim": 128, "window": 0,
         "page": 32, "format": "e4m3", "dtype": "f32", "lens": 3},
        # A batch of verify passes of 1..8 tokens in a sliding layer, unquantised pages; one
        # sequence has nothing cached yet.
        {"name": "verify_pass", "op": "attention", "batch": 32, "q_lo": 1, "q_hi": 8, "kv_lo": 0,
         "kv_hi": 4096, "heads": 8, "kv_heads": 1, "head_dim": 256, "window": 512, "page": 16,
         "format": "bf16", "dtype": "bf16", "lens": 4},
        # Prefill chunks of up to 2048 tokens over up to 8192 cached ones.
        {"name": "chunk_ragged", "op": "attention", "batch": 4, "q_lo": 700, "q_hi": 2048,
         "kv_lo": 3000, "kv_hi": 8192, "heads": 8, "kv_heads": 1, "head_dim": 256, "window": 0,
         "page": 64, "format": "int8", "dtype": "bf16", "lens": 5},
        # One sequence, one drafted token, the engine's vocabulary.
        {"name": "drafts_one", "op": "drafts", "batch": 1, "d_lo": 1, "d_hi": 1, "vocab": 262144,
         "dtype": "f32", "probs": False, "lens": 6},
        # 32 sequences of 0..7 drafted tokens from a prompt lookup, some of them greedy.
        {"name": "drafts_lookup", "op": "drafts", "batch": 32, "d_lo": 0, "d_hi": 7,
         "vocab": 262144, "dtype": "f32", "probs": False, "lens": 7},
        # 48 sequences whose drafter gives probabilities, an odd vocabulary, bf16 logits.
        {"name": "drafts_model", "op": "drafts", "batch": 48, "d_lo": 1, "d_hi": 4,
         "vocab": 100003, "dtype": "bf16", "probs": True, "lens": 8},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["store", "read", "attention", "attention", "attention", "drafts"])
    lens = rng.randrange(1 << 20)
    if op in ("store", "read"):
        c = {"op": op, "kv_heads": rng.choice([1, 2, 8]), "head_dim": rng.choice([64, 128, 256, 512]),
             "page": rng.choice([16, 32, 64, 128]), "format": rng.choice(["bf16", "int8", "e4m3"]),
             "dtype": rng.choice(["f32", "bf16"])}
        most = (16389 if op == "store" else 40001) * 8 * 128 // (c["kv_heads"] * c["head_dim"])
        c["tokens"] = _log(rng, 1, most if c["dtype"] == "bf16" else most // 2)
        c["pages"] = -(-c["tokens"] // c["page"]) + rng.randrange(64)
        return c
    if op == "drafts":
        c = {"op": op, "batch": _log(rng, 1, 32), "d_lo": rng.choice([0, 1]), "d_hi": rng.randint(1, 7),
             "vocab": rng.choice([262144, _log(rng, 1000, 200000)]),
             "dtype": rng.choice(["f32", "bf16"]), "probs": rng.random() < 0.4, "lens": lens}
        if c["probs"]:
            c["d_hi"] = min(c["d_hi"], 4)
            c["batch"] = min(c["batch"], 16)
        return c
    heads, kv_heads = rng.choice([(8, 1), (32, 8), (16, 16), (12, 4), (14, 2)])
    c = {"op": op, "heads": heads, "kv_heads": kv_heads, "head_dim": rng.choice([64, 128, 256, 512]),
         "window": rng.choice([0, 0, 512]), "page": rng.choice([16, 32, 64, 128]),
         "format": rng.choice(["bf16", "int8", "e4m3"]), "dtype": rng.choice(["bf16", "bf16", "f32"]),
         "lens": lens}
    kind = rng.choice(["decode", "verify", "chunk"])
    width = kv_heads * c["head_dim"]
    if kind == "chunk":
        q = _log(rng, 9, 2048)
        batch = rng.randint(1, 4)
        # The score matrix of the plain form and the products' operations bound the context.
        most = min(8192 * 2048 * 4 * 8 // (batch * heads * q),
                   8192 * 2048 * 4 * 8 * 256 // (batch * heads * q * c["head_dim"]), 1 << 26) // 2
        kv = _log(rng, q, max(q, min(most, 65536, 4 * 65537 * 8 * 128 // (batch * width * 2))))
        return {**c, "batch": batch, "q_lo": rng.randint(1, q), "q_hi": q,
                "kv_lo": rng.randint(0, kv), "kv_hi": kv}
    batch = _log(rng, 1, 64)
    q = 1 if kind == "decode" else rng.randint(2, 8)
    most = 4 * 65537 * 8 * 128 // (batch * width * CODE_BYTES[c["format"]])
    kv = _log(rng, 1, min(most, 65537))
    return {**c, "batch": batch, "q_lo": 1, "q_hi": q, "kv_lo": rng.randint(0, kv), "kv_hi": kv}


def _lengths(case):
    """(new tokens, tokens cached including the new ones) of each sequence of an attention case."""
    r = random.Random(case["lens"])
    q = [r.randint(case["q_lo"], case["q_hi"]) for _ in range(case["batch"])]
    kv = [r.randint(case["kv_lo"], case["kv_hi"]) for _ in range(case["batch"])]
    q[0], kv[-1] = case["q_hi"], case["kv_hi"]
    if case["kv_lo"] == 0 and case["batch"] > 1:
        return q, [0] + [max(a, b) for a, b in zip(q[1:], kv[1:])]
    return q, [max(a, b) for a, b in zip(q, kv)]


def _drafts(case):
    r = random.Random(case["lens"])
    d = [r.randint(case["d_lo"], case["d_hi"]) for _ in range(case["batch"])]
    d[-1] = case["d_hi"]
    return d


def work(case):
    if case["op"] in ("store", "read"):
        n = 2 * case["tokens"] * case["kv_heads"] * case["head_dim"]
        io = 4 if case["dtype"] == "f32" else 2
        code = CODE_BYTES[case["format"]]
        scales = 0 if case["format"] == "bf16" else 8 * case["tokens"] * case["kv_heads"]
        once = n * (io + code) + scales + 4 * case["tokens"]
        # A store case stores the rows and reads them back.
        return {"bytes": once * (2 if case["op"] == "store" else 1), "flops": 2 * n}
    if case["op"] == "drafts":
        d, V = _drafts(case), case["vocab"]
        rows = sum(d) + len(d)
        size = 4 if case["dtype"] == "f32" else 2
        # Every row of logits and each sequence's noise are read; of the draft's probabilities at
        # most one row a sequence is (the refused one).
        b = rows * V * size + len(d) * V * 4 + (len(d) * V * 4 if case["probs"] else 0)
        return {"bytes": b, "flops": 5 * rows * V}
    q, kv = _lengths(case)
    H, G, D, W = case["heads"], case["kv_heads"], case["head_dim"], case["window"]
    pairs = tokens = 0
    for n, length in zip(q, kv):
        if length == 0:
            continue
        first = length - n
        tokens += min(length, n + W - 1) if W else length
        if W:
            pairs += sum(min(first + i + 1, W) for i in range(n))
        else:
            pairs += n * first + n * (n + 1) // 2
    io = 4 if case["dtype"] == "f32" else 2
    scale = 0 if case["format"] == "bf16" else 4
    return {"bytes": 2 * tokens * G * (D * CODE_BYTES[case["format"]] + scale) + 2 * sum(q) * H * D * io,
            "flops": 4 * pairs * H * D}


# ------------------------------------------------------------------------------------ inputs

def _rows(g, *shape, dtype):
    """Normalised rows with a few large channels, as keys and values have."""
    x = torch.randn(*shape, generator=g, device="cuda")
    return (x * torch.exp(0.5 * torch.randn(shape[-1], generator=g, device="cuda"))).to(dtype)


def _pool(g, case, pages):
    """A pool whose pages hold quantised rows."""
    shape = (pages, case["kv_heads"], case["page"], case["head_dim"])
    state = {}
    for name in ("k", "v"):
        if case["format"] == "bf16":
            state[name] = torch.randn(*shape, generator=g, device="cuda", dtype=torch.bfloat16)
            state[name + "_scale"] = None
            continue
        if case["format"] == "int8":
            x = torch.randn(*shape, generator=g, device="cuda", dtype=torch.bfloat16)
            state[name] = (x * 36).clamp_(-127, 127).to(torch.int8)
        else:
            x = torch.randn(*shape, generator=g, device="cuda", dtype=torch.bfloat16)
            state[name] = (x * 120).clamp_(-448, 448).to(torch.float8_e4m3fn)
        unit = 1 / 36 if case["format"] == "int8" else 1 / 120
        state[name + "_scale"] = unit * torch.exp(
            0.3 * torch.randn(*shape[:3], generator=g, device="cuda"))
    return state


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    st = {"case": case}
    if case["op"] in ("store", "read"):
        n = case["pages"] * case["page"]
        st.update(_pool(g, case, case["pages"]))
        st["slots"] = torch.randperm(n, generator=g, device="cuda")[:case["tokens"]].to(torch.int32)
        if case["op"] == "store":
            shape = (case["tokens"], case["kv_heads"], case["head_dim"])
            st["new_k"] = _rows(g, *shape, dtype=DTYPES[case["dtype"]])
            st["new_v"] = _rows(g, *shape, dtype=DTYPES[case["dtype"]])
        return st
    if case["op"] == "drafts":
        d = _drafts(case)
        rows, V = sum(d) + len(d), case["vocab"]
        begin = [0]
        for n in d:
            begin.append(begin[-1] + n + 1)
        st["row_begin"] = torch.tensor(begin, dtype=torch.int32, device="cuda")
        # Peaked rows, as a model's are: the drafted token is often the likeliest.
        logits = 2.5 * torch.randn(rows, V, generator=g, device="cuda")
        tokens = torch.randint(0, V, (rows,), generator=g, device="cuda")
        logits[torch.arange(rows, device="cuda"), tokens] += 14 + 4 * torch.rand(
            rows, generator=g, device="cuda")
        # Half of the drafts are the likely token, the others any.
        keep = torch.rand(rows, generator=g, device="cuda") < 0.6
        other = torch.randint(0, V, (rows,), generator=g, device="cuda")
        st["drafts"] = torch.where(keep, tokens, other).to(torch.int32)
        st["logits"] = logits.to(DTYPES[case["dtype"]])
        st["probs"] = None
        if case["probs"]:
            near = logits + 0.7 * torch.randn(rows, V, generator=g, device="cuda")
            st["probs"] = torch.softmax(near, -1)
        st["uniforms"] = torch.rand(rows, generator=g, device="cuda")
        st["gumbel"] = -torch.log(torch.empty(len(d), V, device="cuda").exponential_(generator=g))
        st["temperature"] = torch.tensor([(0.0, 1.0, 0.7, 1.3)[(i + 1) % 4] for i in range(len(d))],
                                         device="cuda")
        return st
    q, kv = _lengths(case)
    page = case["page"]
    need = [-(-n // page) for n in kv]
    spare = 3
    st.update(_pool(g, case, sum(need) + spare))
    order = torch.randperm(sum(need) + spare, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(case["batch"], max(max(need), 1), dtype=torch.int32)
    at = torch.zeros(case["batch"], max(max(need), 1), dtype=torch.int64)
    used = 0
    for b, n in enumerate(need):
        at[b, :n] = torch.arange(used, used + n)
        table[b, :n] = 1
        used += n
    st["page_table"] = torch.where(table.cuda() > 0, order[at.cuda()], torch.zeros_like(order[at.cuda()]))
    begin = [0]
    for n in q:
        begin.append(begin[-1] + n)
    # Rows are scaled so that logits spread over a few units at the operator's scale of 1.
    spread = 1.5 / math.sqrt(case["head_dim"])
    st["q"] = (spread * torch.randn(begin[-1], case["heads"], case["head_dim"], generator=g,
                                    device="cuda")).to(DTYPES[case["dtype"]])
    st["q_begin"] = torch.tensor(begin, dtype=torch.int32, device="cuda")
    st["q_pos"] = torch.tensor([max(0, b - a) for a, b in zip(q, kv)], dtype=torch.int32, device="cuda")
    st["kv_len"] = torch.tensor(kv, dtype=torch.int32, device="cuda")
    st["max_q"], st["max_kv"] = max(q), max(max(kv), 1)
    return st


# ------------------------------------------------------------------------------------ one pass

def run(st):
    return RUN[st["case"]["op"]](st)


def _handle(st):
    return _paged().PagePool(st["k"], st["v"], st["k_scale"], st["v_scale"])


def _plain_quantise(x, fmt):
    """(codes, scale) of rows x [..., D]."""
    if fmt == "bf16":
        return x.to(torch.bfloat16), None
    x = x.float()
    scale = x.abs().amax(-1) / torch.tensor(TOP[fmt], device=x.device)
    r = torch.where(scale[..., None] > 0, x / scale[..., None], torch.zeros_like(x))
    if fmt == "int8":
        return torch.round(r).clamp(-127, 127).to(torch.int8), scale
    return r.clamp(-448, 448).to(torch.float8_e4m3fn), scale


def _plain_store(pages, scales, rows, slots, fmt):
    page = pages.shape[2]
    codes, scale = _plain_quantise(rows, fmt)
    p, o = slots.long() // page, slots.long() % page
    if fmt == "e4m3":
        pages.view(torch.uint8)[p, :, o] = codes.view(torch.uint8)
    else:
        pages[p, :, o] = codes
    if scale is not None:
        scales[p, :, o] = scale


def _plain_read(pages, scales, slots, dtype):
    page = pages.shape[2]
    p, o = slots.long() // page, slots.long() % page
    if pages.dtype == torch.float8_e4m3fn:
        rows = pages.view(torch.uint8)[p, :, o].view(torch.float8_e4m3fn).float()
    else:
        rows = pages[p, :, o].float()
    if scales is not None:
        rows = rows * scales[p, :, o][..., None]
    return rows.to(dtype)


def _run_store(st):
    fmt, dtype = st["case"]["format"], DTYPES[st["case"]["dtype"]]
    if own:
        pool = _handle(st)
        pool.store(st["new_k"], st["new_v"], st["slots"])
        return pool.read(st["slots"], dtype)
    _plain_store(st["k"], st["k_scale"], st["new_k"], st["slots"], fmt)
    _plain_store(st["v"], st["v_scale"], st["new_v"], st["slots"], fmt)
    return (_plain_read(st["k"], st["k_scale"], st["slots"], dtype),
            _plain_read(st["v"], st["v_scale"], st["slots"], dtype))


def _run_read(st):
    dtype = DTYPES[st["case"]["dtype"]]
    if own:
        return _handle(st).read(st["slots"], dtype)
    return (_plain_read(st["k"], st["k_scale"], st["slots"], dtype),
            _plain_read(st["v"], st["v_scale"], st["slots"], dtype))


def _plain_gather(pages, scales, table):
    """[B, KVH, positions, D] in f32."""
    at = table.long()
    if pages.dtype == torch.float8_e4m3fn:
        x = pages.view(torch.uint8)[at].view(torch.float8_e4m3fn).float()
    else:
        x = pages[at].float()
    if scales is not None:
        x = x * scales[at][..., None]
    x = x.transpose(1, 2)
    return x.reshape(x.shape[0], x.shape[1], -1, x.shape[-1])


def _run_attention(st):
    case = st["case"]
    window = case["window"]
    if own:
        return _paged().attention(_handle(st), st["q"], st["q_begin"], st["q_pos"], st["kv_len"],
                                  st["page_table"], st["max_q"], st["max_kv"], window=window)
    q, begin, dev = st["q"], st["q_begin"].long(), st["q"].device
    B, H, G, D = case["batch"], case["heads"], case["kv_heads"], case["head_dim"]
    k = _plain_gather(st["k"], st["k_scale"], st["page_table"])
    v = _plain_gather(st["v"], st["v_scale"], st["page_table"])
    i = torch.arange(st["max_q"], device=dev)
    live = i[None, :] < (begin[1:] - begin[:-1])[:, None]
    row = torch.where(live, begin[:-1, None] + i[None, :], torch.zeros_like(live, dtype=torch.long))
    x = q.float()[row].view(B, st["max_q"], G, H // G, D).permute(0, 2, 3, 1, 4).reshape(B, G, -1, D)
    s = (x @ k.transpose(-1, -2)).view(B, G, H // G, st["max_q"], -1)
    t = torch.arange(k.shape[2], device=dev)
    pos = st["q_pos"].long()[:, None] + i[None, :]
    seen = (t[None, None, :] <= pos[:, :, None]) & (t[None, None, :] < st["kv_len"].long()[:, None, None])
    if window:
        seen &= t[None, None, :] > pos[:, :, None] - window
    s.masked_fill_(~seen[:, None, None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(top > float("-inf"), top, torch.zeros_like(top))).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p.view(B, G, -1, p.shape[-1]) @ v).view(B, G, H // G, st["max_q"], D)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    return o.permute(0, 3, 1, 2, 4).reshape(B, st["max_q"], H, D)[live].to(q.dtype)


def _run_drafts(st):
    case = st["case"]
    most = case["d_hi"]
    if own:
        return _paged().verify_drafts(st["logits"], st["row_begin"], st["drafts"], st["uniforms"],
                                      st["gumbel"], st["temperature"], most, draft_probs=st["probs"])
    begin, dev = st["row_begin"].long(), st["logits"].device
    rows, V = st["logits"].shape
    B = begin.numel() - 1
    r = torch.arange(rows, device=dev)
    seq = torch.searchsorted(begin, r, right=True) - 1
    last = r == begin[seq + 1] - 1
    temp = st["temperature"][seq]
    greedy = temp == 0
    x = st["logits"].float() * torch.where(greedy, torch.ones_like(temp), 1 / temp)[:, None]
    top = x.amax(-1, keepdim=True)
    logp = x - top - (x - top).exp().sum(-1, keepdim=True).log()
    d = st["drafts"].long()
    best = (x == top).to(torch.uint8).argmax(-1)
    q_at = torch.ones_like(temp) if st["probs"] is None else st["probs"][r, d]
    stands = torch.where(greedy, best == d, st["uniforms"] * q_at < logp[r, d].exp()) & ~last
    # Rows before a sequence's first refusal, then that row (or the last one).
    count = torch.zeros(B, dtype=torch.long, device=dev)
    refused = torch.where(~stands, r, torch.full_like(r, rows))
    stop = torch.full((B,), rows, device=dev).scatter_reduce(0, seq, refused, "amin")
    count = stop - begin[:-1]
    drafted = ~last[stop]
    noise = torch.where(greedy[stop][:, None], torch.zeros_like(st["gumbel"]), st["gumbel"])
    key = x[stop] + noise
    left_out = (drafted & ~greedy[stop])[:, None] & (torch.arange(V, device=dev)[None] == d[stop][:, None])
    if st["probs"] is None:
        key = key.masked_fill(left_out, float("-inf"))
    else:
        rest = (logp[stop].exp() - st["probs"][stop]).clamp_min(0)
        some = (drafted & ~greedy[stop])[:, None] & (rest > 0).any(-1, keepdim=True)
        key = torch.where(some, rest.log() + noise, key)
    chosen = (key == key.amax(-1, keepdim=True)).to(torch.uint8).argmax(-1)
    j = torch.arange(most + 1, device=dev)[None]
    at = (begin[:-1, None] + j).clamp_max(rows - 1)
    token = torch.where(j < count[:, None], d[at], torch.where(j == count[:, None], chosen[:, None],
                                                               torch.full_like(at, -1)))
    lp = logp[at, token.clamp_min(0)]
    return (token.to(torch.int32), torch.where(token >= 0, lp, torch.zeros_like(lp)),
            (count + 1).to(torch.int32))


RUN = {"store": _run_store, "read": _run_read, "attention": _run_attention, "drafts": _run_drafts}


# ------------------------------------------------------------------------------------ 64 bits

def _exact_rows(pages, scales, page_ids, offsets):
    """Rows [n, KVH, D] in 64 bits."""
    raw = pages.view(torch.uint8) if pages.dtype == torch.float8_e4m3fn else pages
    x = raw[page_ids, :, offsets]
    if pages.dtype == torch.float8_e4m3fn:
        x = x.contiguous().view(torch.float8_e4m3fn)
    x = x.double()
    return x if scales is None else x * scales[page_ids, :, offsets].double().unsqueeze(-1)


def _exact_quantised(rows, fmt):
    """What rows stand for once they are stored, in 64 bits."""
    x = rows.double()
    if fmt == "bf16":
        return rows.to(torch.bfloat16).double()
    s = (x.abs().max(dim=-1, keepdim=True).values / TOP[fmt]).clamp_min(1e-300)
    y = x / s
    if fmt == "int8":
        return torch.round(y) * s
    # e4m3: 3 fraction bits, exponents from -6.
    unit = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(1e-30))).clamp_min(-6) - 3)
    return torch.round(y / unit) * unit * s


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "store":
        return [_exact_quantised(st["new_k"], case["format"]), _exact_quantised(st["new_v"], case["format"])]
    if case["op"] == "read":
        s = st["slots"].long()
        return [_exact_rows(st[n], st[n + "_scale"], s // case["page"], s % case["page"]) for n in ("k", "v")]
    if case["op"] == "attention":
        q, kv = _lengths(case)
        H, G = case["heads"], case["kv_heads"]
        out = torch.zeros(*st["q"].shape, dtype=torch.float64, device="cuda")
        row = 0
        for b, (n, length) in enumerate(zip(q, kv)):
            if length:
                t = torch.arange(length, device="cuda")
                ids = st["page_table"][b].long()[t // case["page"]]
                k = _exact_rows(st["k"], st["k_scale"], ids, t % case["page"])
                v = _exact_rows(st["v"], st["v_scale"], ids, t % case["page"])
                where = length - n + torch.arange(n, device="cuda")
                hidden = t[None] > where[:, None]
                if case["window"]:
                    hidden |= t[None] <= where[:, None] - case["window"]
                for h in range(H):
                    c = h // (H // G)
                    z = st["q"][row:row + n, h].double() @ k[:, c].T
                    z[hidden] = -math.inf
                    out[row:row + n, h] = torch.softmax(z, dim=1) @ v[:, c]
            row += n
        return out
    tokens, lp, counts = [], [], []
    begin = st["row_begin"].tolist()
    for b in range(case["batch"]):
        T = st["temperature"][b].double().item()
        lps = [0.0] * (case["d_hi"] + 1)
        for j, r in enumerate(range(begin[b], begin[b + 1])):
            x = st["logits"][r].double() / (T or 1.0)
            logp = x - torch.logsumexp(x, 0)
            d = int(st["drafts"][r])
            end = r == begin[b + 1] - 1
            if not end:
                u = st["uniforms"][r].double().item()
                w = 1.0 if st["probs"] is None else st["probs"][r, d].double().item()
                if (int(x.argmax()) == d) if T == 0 else (u * w < math.exp(logp[d].item())):
                    lps[j] = logp[d].item()
                    continue
            g = st["gumbel"][b].double() if T else torch.zeros_like(x)
            key = x + g
            if not end and T:
                if st["probs"] is None:
                    key[d] = -math.inf
                else:
                    rest = (logp.exp() - st["probs"][r].double()).clamp_min(0)
                    if bool((rest > 0).any()):
                        key = rest.log() + g
            lps[j] = logp[int(key.argmax())].item()
            break
        lp.append(lps)
    return [None, torch.tensor(lp, dtype=torch.float64), None]
