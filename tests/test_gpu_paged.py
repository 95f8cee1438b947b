"""The paged-cache operators (g4_op_page_store / page_read / paged_attention / verify_drafts)
against their definitions in 64 bits, at the sizes and masks where they can go wrong.

Tolerances. Stored codes and what is read back are exact: the same f32 operations in the same
order. Attention, with A = max_t scale * sum_d |q_d k_td| of the row and B_d = sum_t p_t |v_td|:
scores accumulate exact products in f32, so a score is off by at most 2^-21 A and its weight by as
much relatively; bf16 rows add the rounding of the result (2^-8, bf16's unit roundoff: 1 + 2^-8
rounds to 1) and of the weights (2^-8 each in bf16 pages, whose products are bf16, 2^-11 in 8-bit
pages, whose products are f16); f32 rows carry q and the weights in parts of at least 22 bits together. Weights are held relative to
the largest of their row in a type with a smallest step: F bounds what n of them below that step
add, 2^-126 of the largest for bf16 pages (f32's exponents) and 2^-38 for 8-bit pages (f16 parts
scaled by 2^14), which shows only where the heavy positions' codes are zero; results below the
smallest normal number of their type, 2^-126, may be rounded to zero. Draft log probabilities:
f32 sums of exps, 2^-20 of the terms, plus one rounding of values below 2^6 in magnitude.
"""
from __future__ import annotations

import importlib
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

HEAD_DIMS = [64, 128, 256, 512]
FORMATS = ["bf16", "int8", "e4m3"]


@pytest.fixture(scope="module")
def paged(pkg, cuda):
    return importlib.import_module(pkg.__name__ + ".paged")


@pytest.fixture(autouse=True)
def _no_flags(paged):
    paged.errors()
    yield
    assert paged.errors() == 0


def gen(torch, seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def make_pool(paged, torch, fmt, pages, page, heads, hd, seed=1, unit=0.03):
    """A pool of random rows (values of a few units)."""
    pool = paged.PagePool.create(pages, page, heads, hd, fmt)
    g = gen(torch, seed)
    for x, s in ((pool.k, pool.k_scale), (pool.v, pool.v_scale)):
        if fmt == "bf16":
            x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
            continue
        if fmt == "int8":
            x.copy_(torch.randint(-127, 128, x.shape, generator=g, device="cuda").to(torch.int8))
        else:
            x.copy_((torch.randn(x.shape, generator=g, device="cuda") * 60).clamp(-448, 448).to(torch.float8_e4m3fn))
        s.copy_(unit * torch.exp(torch.randn(s.shape, generator=g, device="cuda")))
    return pool


def values(pool, torch):
    """k, v [n_pages, kv_heads, page, hd] in 64 bits."""
    out = []
    for x, s in ((pool.k, pool.k_scale), (pool.v, pool.v_scale)):
        x = x.float().double()
        out.append(x if s is None else x * s.double()[..., None])
    return out


# ------------------------------------------------------------------------------ store and read

def quantise(np_rows, fmt, torch):
    """(codes as f32 values, scales) of f32 rows by the definition, in numpy's f32."""
    x = np_rows.astype(np.float32)
    if fmt == "bf16":
        return torch.from_numpy(x).to(torch.bfloat16).float().numpy(), None
    top = np.float32(127.0 if fmt == "int8" else 448.0)
    amax = np.abs(x).max(-1)
    s = (amax / top).astype(np.float32)
    with np.errstate(all="ignore"):
        r = np.where(s[..., None] > 0, x / s[..., None], np.float32(0))
    if fmt == "int8":
        c = np.clip(np.rint(r), -127, 127)
    else:
        c = torch.from_numpy(np.clip(r, -448, 448)).to(torch.float8_e4m3fn).float().numpy()
    bad = ~np.isfinite(x).all(-1)
    s = np.where(bad, np.float32(np.nan), s)
    return np.where(bad[..., None], 0, c).astype(np.float32), s


@pytest.mark.parametrize("hd", HEAD_DIMS)
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype,tokens,heads,page", [("f32", 37, 1, 16), ("bf16", 1, 3, 64), ("bf16", 200, 8, 48)])
def test_store_and_read_exact(paged, cuda, hd, fmt, dtype, tokens, heads, page):
    torch = cuda
    pages = -(-tokens // page) + 3
    pool = make_pool(paged, torch, fmt, pages, page, heads, hd)
    before = [t.clone() for t in (pool.k, pool.v)]
    g = gen(torch, 5)
    t = {"f32": torch.float32, "bf16": torch.bfloat16}[dtype]
    # Rows of one packed projection: K and V are slices with a longer token stride.
    packed = (torch.randn(tokens, 2 * heads + 1, hd, generator=g, device="cuda") * 3).to(t)
    k, v = packed[:, :heads], packed[:, heads + 1:]
    k[0, 0] = 0                              # an all-zero row
    v[-1, -1] = 1e-41 if dtype == "f32" else 0   # a row whose scale is subnormal or zero
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens].to(torch.int32)
    pool.store(k, v, slots)
    kr, vr = pool.read(slots, torch.float32)
    kb, vb = pool.read(slots, torch.bfloat16)
    for rows, f32, b16, pages_t, scales, old in ((k, kr, kb, pool.k, pool.k_scale, before[0]),
                                                 (v, vr, vb, pool.v, pool.v_scale, before[1])):
        codes, s = quantise(rows.float().cpu().numpy(), fmt, torch)
        p, o = (slots // page).long(), (slots % page).long()
        raw = pages_t.view(torch.uint8) if fmt == "e4m3" else pages_t
        got = raw[p, :, o]
        got = got.contiguous().view(torch.float8_e4m3fn) if fmt == "e4m3" else got
        np.testing.assert_array_equal(got.float().cpu().numpy(), codes)
        want = codes if s is None else codes * s[..., None]
        if s is not None:
            np.testing.assert_array_equal(scales[p, :, o].cpu().numpy(), s)
        np.testing.assert_array_equal(f32.cpu().numpy(), want)
        np.testing.assert_array_equal(b16.float().cpu().numpy(), torch.from_numpy(want).to(torch.bfloat16).float().numpy())
        # Every other position keeps what it held.
        keep = torch.ones(pages * page, dtype=torch.bool, device="cuda")
        keep[slots.long()] = False
        keep = keep.view(pages, page)
        a = raw.transpose(1, 2)[keep]
        b = (old.view(torch.uint8) if fmt == "e4m3" else old).transpose(1, 2)[keep]
        assert torch.equal(a, b)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_store_marks_rows_that_are_not_finite(paged, cuda, fmt, bad):
    torch = cuda
    pool = paged.PagePool.create(2, 16, 2, 128, fmt)
    k = torch.randn(3, 2, 128, generator=gen(torch, 2), device="cuda")
    k[1, 1, 77] = bad
    slots = torch.tensor([3, 20, 9], dtype=torch.int32, device="cuda")
    pool.store(k, k, slots)
    kr, vr = pool.read(slots)
    want = torch.zeros(3, 2, dtype=torch.bool, device="cuda")
    want[1, 1] = True
    for r in (kr, vr):
        assert torch.equal(r.isnan().all(-1), want) and torch.equal(r.isnan().any(-1), want)


def test_slots_skipped_and_reported(paged, cuda):
    torch = cuda
    pool = make_pool(paged, torch, "int8", 2, 16, 1, 64)
    old = pool.k.clone()
    k = torch.ones(3, 1, 64, device="cuda")
    pool.store(k, k, torch.tensor([-1, 7, -5], dtype=torch.int32, device="cuda"))
    assert torch.equal(pool.k[0, 0, 7].float(), torch.full((64,), 127.0, device="cuda"))
    old[0, 0, 7] = pool.k[0, 0, 7]
    assert torch.equal(pool.k, old)
    assert paged.errors() == 0
    pool.store(k, k, torch.tensor([32, -1, 2**31 - 1], dtype=torch.int32, device="cuda"))
    assert torch.equal(pool.k, old)
    assert paged.errors() == paged.BAD_PAGE
    kr, _ = pool.read(torch.tensor([32, -1, 7], dtype=torch.int32, device="cuda"))
    assert paged.errors() == paged.BAD_PAGE
    assert torch.equal(kr[:2], torch.zeros(2, 1, 64, device="cuda")) and torch.allclose(kr[2], torch.ones(1, 64, device="cuda"))
    assert pool.read(torch.empty(0, dtype=torch.int32, device="cuda"))[0].shape == (0, 1, 64)


# ------------------------------------------------------------------------------ attention

def layout(torch, kv, page, extra, seed):
    """(page table, pages): pages in a random order, entries past a sequence's last page -1."""
    need = [-(-n // page) for n in kv]
    total = sum(need) + extra
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.full((len(kv), max(max(need), 1)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table.cuda(), total


def reference(torch, pool, q, spans, table, window, scale):
    """(out, lse, A, B, F) in 64 bits; spans: (row, n, pos, kv) per sequence."""
    kk, vv = values(pool, torch)
    rows, H, D = q.shape
    G = pool.kv_heads
    out = torch.zeros(rows, H, D, dtype=torch.float64, device="cuda")
    lse = torch.full((rows, H), -math.inf, dtype=torch.float64, device="cuda")
    A = torch.zeros(rows, H, 1, dtype=torch.float64, device="cuda")
    B = torch.zeros_like(out)
    F = torch.zeros_like(A)
    top = torch.full_like(pool.v[:, :, :, 0], 1, dtype=torch.float64)
    step = 2.0 ** -126
    if pool.v_scale is None:
        top *= pool.v.double().abs().amax(-1)
    else:
        top *= pool.v_scale.double() * (127 if pool.v.dtype == torch.int8 else 448)
        step = 2.0 ** -38
    for b, (row, n, pos, kv) in enumerate(spans):
        if n == 0 or kv == 0:
            continue
        t = torch.arange(kv, device="cuda")
        # Only pages with a visible position have an entry.
        ids = table[b].long()[t // pool.page_size].clamp_min(0)
        k, v = kk[ids, :, t % pool.page_size], vv[ids, :, t % pool.page_size]
        p = pos + torch.arange(n, device="cuda")
        see = t[None] <= p[:, None]
        if window:
            see &= t[None] > p[:, None] - window
        some = see.any(-1)
        for h in range(H):
            c = h // (H // G)
            x = q[row:row + n, h].double()
            # A position no row sees may hold anything.
            kc = torch.where(see.any(0)[:, None], k[:, c], torch.zeros_like(k[:, c]))
            vc = torch.where(see.any(0)[:, None], v[:, c], torch.zeros_like(v[:, c]))
            s = (scale * (x @ kc.T)).masked_fill(~see, -math.inf)
            w = torch.where(some[:, None], torch.softmax(s, -1), torch.zeros_like(s))
            out[row:row + n, h] = w @ vc
            lse[row:row + n, h] = torch.where(some, torch.logsumexp(s, -1), lse[row:row + n, h])
            A[row:row + n, h, 0] = (abs(scale) * (x.abs() @ kc.abs().T)).masked_fill(~see, 0).amax(-1)
            B[row:row + n, h] = w @ vc.abs()
            each = torch.where(see.any(0), top[ids, c, t % pool.page_size], torch.zeros_like(t, dtype=torch.float64))
            F[row:row + n, h, 0] = kv * step * (w * each).amax(-1)
    return out, lse, A, B, F


def check(torch, got, glse, want, lse, A, B, F, bf16, pages16=False):
    tol = (2.0 ** -21 * 2 * A + (2.0 ** -8 + 2.0 ** -11 + (2.0 ** -8 if pages16 else 0) if bf16 else 2.0 ** -19)) * B + F + 2.0 ** -126
    off = (got.double() - want).abs()
    assert not got.isnan().any()
    bad = off > tol
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} off, worst {float((off / tol.clamp_min(1e-300)).max()):.3g} "
                           f"tolerances, first at {bad.nonzero()[0].tolist()}")
    if glse is not None:
        fin = lse.isfinite()
        assert torch.equal(fin, glse.isfinite()) and (glse[~fin] == -math.inf).all()
        d = (glse.double() - lse)[fin].abs()
        assert (d <= (2.0 ** -20 * A[..., 0][fin] + 2.0 ** -18 * (1 + lse[fin].abs()))).all(), float(d.max())


def run_case(paged, torch, q_len, kv, heads, kv_heads, hd, page, fmt, dtype, window=0, scale=None, seed=3,
             pos=None, gap=0, poison=True, spread=1.5, max_q=None, max_kv=None):
    """A ragged batch through paged.attention against the reference. Positions that no row sees
    hold NaN (through the scale of 8-bit pages) where `poison`."""
    g = gen(torch, seed)
    table, pages = layout(torch, kv, page, 2, seed)
    pool = make_pool(paged, torch, fmt, pages, page, kv_heads, hd, seed)
    begin = [gap]
    for n in q_len:
        begin.append(begin[-1] + n)
    rows = begin[-1] + gap
    t = {"f32": torch.float32, "bf16": torch.bfloat16}[dtype]
    unit = 1.0 if fmt == "bf16" else (2.2 if fmt == "int8" else 1.8) * 1.6
    scale = spread / math.sqrt(hd) / unit if scale is None else scale
    q = torch.randn(rows, heads, hd, generator=g, device="cuda").to(t)
    pos = [n - m for m, n in zip(q_len, kv)] if pos is None else pos
    spans = [(begin[b], q_len[b], pos[b], kv[b]) for b in range(len(kv))]
    if poison:
        seen = torch.zeros(pages, page, dtype=torch.bool)
        tb = table.cpu()
        for b, (_, n, p, length) in enumerate(spans):
            if n == 0:
                continue
            lo = max(0, p - window + 1) if window else 0
            for x in range(lo, min(p + n, length)):
                seen[tb[b, x // page], x % page] = True
            if window:   # freed pages below the window
                table[b, :lo // page] = -1
        for x, s in ((pool.k, pool.k_scale), (pool.v, pool.v_scale)):
            if s is None:
                x.transpose(1, 2)[~seen.cuda()] = float("nan")
            else:
                s.transpose(1, 2)[~seen.cuda()] = float("nan")
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    lse = torch.full((rows, heads), 7.0, device="cuda")
    out = torch.full((rows, heads, hd), 7.0, device="cuda", dtype=t)
    paged.attention(pool, q, ints(begin), ints(pos), ints(kv), table, max_q or max(q_len + [1]),
                    max_kv or max(kv + [1]), window=window, scale=scale, out=out, lse=lse)
    want, wl, A, B, F = reference(torch, pool, q, spans, table, window, scale)
    for a, b in ((0, gap), (rows - gap, rows)):   # rows of no sequence stay as they were
        assert (out[a:b] == 7).all() and (lse[a:b] == 7).all()
    sl = slice(gap, rows - gap)
    check(torch, out[sl], lse[sl], want[sl], wl[sl], A[sl], B[sl], F[sl], dtype == "bf16", fmt == "bf16")
    return out


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("hd", HEAD_DIMS)
def test_decode_ragged(paged, cuda, hd, fmt, dtype):
    run_case(paged, cuda, [1, 1, 0, 1, 1], [1, 17, 5, 300, 128], 8, 1, hd, 16, fmt, dtype, gap=2)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 4), (14, 2), (24, 1), (32, 8), (128, 1)])
def test_head_groups(paged, cuda, heads, kv_heads):
    run_case(paged, cuda, [1, 1, 2], [70, 33, 260], heads, kv_heads, 128, 32, "int8", "bf16")
    run_case(paged, cuda, [40, 5], [70, 133], heads, kv_heads, 64, 32, "e4m3", "f32")


@pytest.mark.parametrize("window", [1, 7, 16, 128, 512])
@pytest.mark.parametrize("fmt,dtype", [("int8", "bf16"), ("bf16", "bf16"), ("e4m3", "f32")])
def test_windows_read_only_their_pages(paged, cuda, window, fmt, dtype):
    run_case(paged, cuda, [1, 3, 20, 150], [600, 1000, 700, 150], 8, 1, 256, 64, fmt, dtype, window=window)


@pytest.mark.parametrize("fmt,dtype", [("int8", "bf16"), ("bf16", "bf16"), ("e4m3", "f32"), ("bf16", "f32")])
def test_rows_that_see_nothing(paged, cuda, fmt, dtype):
    # Nothing cached; a window that lies past the cache; rows before position 0; a normal one.
    run_case(paged, cuda, [2, 3, 4, 2], [0, 40, 30, 9], 8, 2, 128, 16, fmt, dtype, window=8, pos=[0, 60, -2, 7])
    run_case(paged, cuda, [1], [0], 8, 1, 64, 16, fmt, dtype, pos=[0])


@pytest.mark.parametrize("page", [16, 48, 64, 112, 128, 1024])
def test_page_sizes(paged, cuda, page):
    run_case(paged, cuda, [1, 1, 4], [2 * page + 1, page, page + 7], 8, 1, 256, page, "int8", "bf16")
    run_case(paged, cuda, [70, 33], [2 * page + 100, page + 40], 8, 1, 128, page, "bf16", "bf16")


@pytest.mark.parametrize("n", [2, 3, 5, 8, 9, 16, 17, 31])
@pytest.mark.parametrize("fmt,dtype,hd", [("int8", "bf16", 256), ("bf16", "bf16", 512), ("e4m3", "f32", 128)])
def test_verify_widths(paged, cuda, n, fmt, dtype, hd):
    run_case(paged, cuda, [n, 1, max(1, n - 1)], [n + 500, 77, n], 8, 1, hd, 32, fmt, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("hd", HEAD_DIMS)
def test_chunks(paged, cuda, hd, fmt, dtype):
    run_case(paged, cuda, [129, 1, 300, 64], [129, 40, 700, 1000], 8, 1, hd, 64, fmt, dtype, gap=1)


def test_chunk_of_many_heads_without_cache(paged, cuda):
    run_case(paged, cuda, [257, 100], [257, 100], 12, 4, 128, 16, "e4m3", "bf16")


@pytest.mark.parametrize("fmt,dtype,hd", [("int8", "bf16", 256), ("e4m3", "f32", 64), ("bf16", "bf16", 512)])
def test_long_context_split(paged, cuda, fmt, dtype, hd):
    run_case(paged, cuda, [1, 1], [20011, 9000], 8, 1, hd, 64, fmt, dtype)
    run_case(paged, cuda, [5], [12345], 8, 2, hd, 64, fmt, dtype)


@pytest.mark.parametrize("q_len", [[1, 1], [40, 3]])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_scales_of_any_magnitude(paged, cuda, fmt, q_len):
    """V scales from 1e-30 to 1e20 and all-zero rows in one context, scores far apart."""
    torch = cuda
    kv = [300, 64]
    table, pages = layout(torch, kv, 16, 1, 4)
    pool = make_pool(paged, torch, fmt, pages, 16, 1, 128, 4)
    g = gen(torch, 9)
    pool.v_scale.copy_(torch.exp(torch.empty_like(pool.v_scale).uniform_(-69, 46, generator=g)))
    pool.v_scale[torch.rand(pool.v_scale.shape, generator=g, device="cuda") < 0.2] = 0
    rows = sum(q_len)
    q = torch.randn(rows, 8, 128, generator=g, device="cuda").bfloat16()
    begin, pos = [0, q_len[0], rows], [kv[0] - q_len[0], kv[1] - q_len[1]]
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    lse = torch.empty(rows, 8, device="cuda")
    out = paged.attention(pool, q, ints(begin), ints(pos), ints(kv), table, max(q_len), 300, scale=0.3, lse=lse)
    spans = [(begin[b], q_len[b], pos[b], kv[b]) for b in range(2)]
    check(torch, out, lse, *reference(torch, pool, q, spans, table, 0, 0.3), True)


@pytest.mark.parametrize("q_len", [1, 40])
def test_scores_beyond_exp_range(paged, cuda, q_len):
    """Scores of thousands: the running maximum carries them; the likeliest position wins alone."""
    run_case(paged, cuda, [q_len], [200], 8, 1, 64, 16, "int8", "bf16", spread=300.0)
    run_case(paged, cuda, [q_len], [200], 8, 1, 64, 16, "bf16", "bf16", scale=0.0)
    run_case(paged, cuda, [q_len], [200], 8, 1, 64, 16, "e4m3", "f32", scale=-0.2)


@pytest.mark.parametrize("q_len", [1, 33])
@pytest.mark.parametrize("mag", [1e-30, 1e30])
def test_f32_queries_of_any_magnitude(paged, cuda, q_len, mag):
    torch = cuda
    table, pages = layout(torch, [90], 16, 1, 4)
    pool = make_pool(paged, torch, "int8", pages, 16, 1, 64, 4)
    q = torch.randn(q_len, 8, 64, generator=gen(torch, 9), device="cuda") * mag
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    out = paged.attention(pool, q, ints([0, q_len]), ints([90 - q_len]), ints([90]), table, q_len, 90, scale=0.1 / mag)
    want = reference(torch, pool, q, [(0, q_len, 90 - q_len, 90)], table, 0, float(np.float32(0.1 / mag)))
    check(torch, out, None, *want, False)


def test_strided_rows_and_another_stream(paged, cuda):
    torch = cuda
    table, pages = layout(torch, [77, 300], 16, 1, 4)
    pool = make_pool(paged, torch, "int8", pages, 16, 2, 128, 4)
    packed = torch.randn(3, 12, 128, generator=gen(torch, 9), device="cuda").bfloat16()
    q = packed[:, 2:10]
    wide = torch.full((3, 9, 128), 3.0, device="cuda", dtype=torch.bfloat16)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    args = (ints([0, 1, 3]), ints([76, 298]), ints([77, 300]), table, 2, 300)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        paged.attention(pool, q, *args, scale=0.05, out=wide[:, :8])
    side.synchronize()
    assert (wide[:, 8] == 3).all()
    spans = [(0, 1, 76, 77), (1, 2, 298, 300)]
    check(torch, wide[:, :8], None, *reference(torch, pool, q, spans, table, 0, float(np.float32(0.05))), True)
    again = paged.attention(pool, q, *args, scale=0.05)
    assert torch.equal(again, wide[:, :8])


def test_repeated_calls_are_bit_identical_and_leave_the_workspace_ready(paged, cuda):
    outs = [run_case(paged, cuda, [1, 1, 6], [5000, 300, 900], 8, 1, 256, 64, "int8", "bf16") for _ in range(3)]
    run_case(paged, cuda, [1] * 9, [64 * i + 1 for i in range(9)], 16, 16, 64, 16, "bf16", "f32")
    outs.append(run_case(paged, cuda, [1, 1, 6], [5000, 300, 900], 8, 1, 256, 64, "int8", "bf16"))
    assert all(cuda.equal(o, outs[0]) for o in outs)


def test_attention_in_a_graph(paged, cuda):
    torch = cuda
    table, pages = layout(torch, [600], 16, 1, 4)
    pool = make_pool(paged, torch, "e4m3", pages, 16, 1, 256, 4)
    q = torch.randn(1, 8, 256, generator=gen(torch, 9), device="cuda").bfloat16()
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    begin, pos, kv = ints([0, 1]), ints([599]), ints([600])
    out = torch.empty_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):   # warm-up: the stream's workspace exists before the capture
        paged.attention(pool, q, begin, pos, kv, table, 1, 600, out=out)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            paged.attention(pool, q, begin, pos, kv, table, 1, 600, out=out)
    for n in (600, 77):
        pos.fill_(n - 1)
        kv.fill_(n)
        graph.replay()
        torch.cuda.synchronize()
        check(torch, out, None, *reference(torch, pool, q, [(0, 1, n - 1, n)], table, 0, 1.0), True)


@pytest.mark.parametrize("q_len", [1, 40])
def test_bad_pages_and_lengths_are_reported(paged, cuda, q_len):
    torch = cuda
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    table, pages = layout(torch, [100], 16, 1, 4)
    pool = make_pool(paged, torch, "int8", pages, 16, 1, 64, 4)
    q = torch.randn(q_len, 8, 64, generator=gen(torch, 9), device="cuda").bfloat16()
    base = (ints([0, q_len]), ints([100 - q_len]), ints([100]))
    good = paged.attention(pool, q, *base, table, q_len, 100, scale=0.1)
    for bad in (pages, -1, 2**31 - 1):
        t = table.clone()
        t[0, 2] = bad
        out = paged.attention(pool, q, *base, t, q_len, 100, scale=0.1)
        assert out.isfinite().all() and paged.errors() == paged.BAD_PAGE
    # A cache longer than the bound is cut off at it.
    cut = paged.attention(pool, q, base[0], base[1], ints([5000]), table, q_len, 100, scale=0.1)
    assert paged.errors() == paged.BAD_LENGTH
    assert torch.equal(cut, good)
    paged.attention(pool, q, ints([0, q_len + 5]), *base[1:], table, q_len, 100, scale=0.1)
    assert paged.errors() == paged.BAD_LENGTH


# ------------------------------------------------------------------------------ drafts

def verify_reference(logits, begin, drafts, probs, u, gumbel, temp, width):
    """The definition in numpy, 64 bits; also the smallest margin of any decision."""
    B = len(begin) - 1
    tokens, lps, counts, margin = np.full((B, width), -1), np.zeros((B, width)), np.zeros(B, int), math.inf
    for b in range(B):
        n = begin[b + 1] - begin[b]
        if n == 0:
            continue
        T = temp[b]
        for j in range(n):
            r = begin[b] + j
            x = logits[r].astype(np.float64)
            if T != 0:
                x = x * np.float64(np.float32(1) / np.float32(T))
            top = x.max()
            logp = x - top - np.log(np.exp(x - top).sum())
            d, drafted = int(drafts[r]), j < n - 1
            if drafted:
                if T == 0:
                    ok = int(np.argmax(x)) == d
                else:
                    w = 1.0 if probs is None else float(probs[r, d]) if 0 <= d < x.size else 1.0
                    p = math.exp(logp[d]) if 0 <= d < x.size else -1.0
                    ok = u[r] * w < p
                    margin = min(margin, abs(u[r] * w - p) / max(abs(p), 1e-9))
                if ok:
                    tokens[b, j], lps[b, j] = d, logp[d]
                    continue
            key = x + (0 if T == 0 else gumbel[b].astype(np.float64))
            if drafted and T != 0:
                if probs is None:
                    if 0 <= d < x.size:
                        key[d] = -np.inf
                else:
                    left = np.maximum(np.exp(logp) - probs[r], 0)
                    if (left > 0).any():
                        with np.errstate(divide="ignore"):
                            key = np.log(left) + gumbel[b]
            pick = int(np.argmax(key))
            two = np.partition(key[np.isfinite(key)], -2)[-2:] if np.isfinite(key).sum() > 1 else np.array([0, 1])
            if T != 0:
                margin = min(margin, two[1] - two[0])
            tokens[b, j], lps[b, j], counts[b] = pick, logp[pick], j + 1
            break
    return tokens, lps, counts, margin


@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("dtype,vocab,lens", [
    ("f32", 4096, [1, 3, 0, 5, 2, 2]), ("f32", 1, [1, 2]), ("f32", 33, [4, 4, 4]), ("bf16", 50001, [2, 5, 1]),
    ("bf16", 40960, [3, 3]), ("f32", 262144, [2]), ("f32", 20001, [8] * 6),
])
def test_verify_drafts(paged, cuda, probs, dtype, vocab, lens):
    torch = cuda
    rng = np.random.default_rng(vocab + 7 * len(lens) + probs)
    begin = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    rows, B = int(begin[-1]), len(lens)
    logits = (2.0 * rng.standard_normal((rows, vocab))).astype(np.float32)
    hot = rng.integers(0, vocab, rows)
    logits[np.arange(rows), hot] += 9 + 4 * rng.random(rows)
    t = torch.from_numpy(logits).cuda().to({"f32": torch.float32, "bf16": torch.bfloat16}[dtype])
    logits = t.float().cpu().numpy()
    drafts = np.where(rng.random(rows) < 0.75, hot, rng.integers(0, vocab, rows)).astype(np.int32)
    q = None
    if probs:
        z = logits + 0.8 * rng.standard_normal((rows, vocab))
        q = np.exp(z - z.max(-1, keepdims=True))
        q = (q / q.sum(-1, keepdims=True)).astype(np.float32)
    u = rng.random(rows).astype(np.float32)
    gum = -np.log(rng.exponential(size=(B, vocab))).astype(np.float32)
    temp = np.array([(1.0, 0.7, 0.0, 1.4)[i % 4] for i in range(B)], np.float32)
    width = max(lens)
    cu = lambda a: torch.from_numpy(a).cuda()
    tokens, lp, counts = paged.verify_drafts(t, cu(begin), cu(drafts), cu(u), cu(gum), cu(temp), width - 1,
                                             draft_probs=None if q is None else cu(q))
    wt, wl, wc, margin = verify_reference(logits, begin, drafts, q, u, gum, temp, width)
    assert margin > 1e-5, "the inputs leave a decision to rounding"
    np.testing.assert_array_equal(counts.cpu().numpy(), wc)
    np.testing.assert_array_equal(tokens.cpu().numpy(), wt)
    np.testing.assert_allclose(lp.cpu().numpy(), wl, rtol=2.0 ** -20, atol=2.0 ** -17)


def small_verify(paged, torch, logits, drafts, u, gumbel, temp, probs=None, begin=None, most=None):
    cu = lambda a, t: torch.tensor(a, dtype=t, device="cuda")
    begin = [0, len(logits)] if begin is None else begin
    tokens, lp, counts = paged.verify_drafts(
        cu(logits, torch.float32), cu(begin, torch.int32), cu(drafts, torch.int32), cu(u, torch.float32),
        cu(gumbel, torch.float32), cu(temp, torch.float32), len(logits) - 1 if most is None else most,
        draft_probs=None if probs is None else cu(probs, torch.float32))
    return tokens.tolist(), lp.tolist(), counts.tolist()


def test_verify_ties_masks_and_odd_values(paged, cuda):
    torch = cuda
    inf, nan = math.inf, math.nan
    # Greedy ties go to the lowest token; a draft equal to another of the tied ones is refused.
    assert small_verify(paged, torch, [[1, 5, 5, 0], [2, 2, 2, 2]], [2, 0], [0, 0], [[0] * 4], [0.0])[0] == [[1, -1]]
    assert small_verify(paged, torch, [[1, 5, 5, 0], [2, 2, 2, 2]], [1, 0], [0, 0], [[0] * 4], [0.0])[0] == [[1, 0]]
    # Masked tokens (-inf) are never emitted, a masked draft never stands, even at u = 0.
    t, lp, c = small_verify(paged, torch, [[-inf, 0, -inf, 0], [0] * 4], [0, 0], [0.0, 0.0], [[9, 0, 9, 1]], [1.0])
    assert t == [[3, -1]] and c == [1] and abs(lp[0][0] + math.log(2)) < 1e-6
    # Drafts outside the vocabulary are refused and leave the race whole.
    for d in (-1, 4, 2**31 - 1):
        assert small_verify(paged, torch, [[0, 3, 0, 0], [0] * 4], [d, 0], [0.0, 0.0], [[0] * 4], [1.0])[0] == [[1, -1]]
    # A NaN is not the greatest; its row's probabilities are NaN and no draft of it stands.
    t, lp, c = small_verify(paged, torch, [[0, nan, 2, 0], [0] * 4], [2, 0], [0.0, 0.0], [[0] * 4], [1.0])
    assert t == [[0, -1]] and math.isnan(lp[0][0])
    # Everything masked: the lowest token.
    assert small_verify(paged, torch, [[-inf] * 4], [0], [0.0], [[0] * 4], [1.0])[0] == [[0]]
    # q equal to p: no remainder, the draft refused by u = 1 is followed by a sample of p.
    p = [0.5, 0.25, 0.125, 0.125]
    t, _, c = small_verify(paged, torch, [[math.log(x) + 1 for x in p], [0] * 4], [1, 0], [1.5, 0], [[0, 0, 5, 0]],
                           [1.0], probs=[[2.0] * 4, p])
    assert t == [[2, -1]]


def test_verify_cuts_off_long_sequences(paged, cuda):
    torch = cuda
    t, _, c = small_verify(paged, torch, [[0, 9]] * 4, [1] * 4, [0.0] * 4, [[0, 0]], [1.0], most=2)
    assert t == [[1, 1, 1]] and c == [3]
    assert paged.errors() == paged.BAD_LENGTH


def test_sampling_follows_the_target(paged, cuda):
    """Whatever the drafter proposes, the emitted token follows p: 40,000 one-draft sequences over
    a vocabulary of 6, each frequency within 5 standard deviations."""
    torch = cuda
    B, V = 40000, 6
    g = gen(torch, 31)
    row = torch.tensor([1.0, 0.2, -0.5, 2.0, 0.0, -3.0], device="cuda")
    logits = row.expand(2 * B, V).contiguous()
    begin = torch.arange(0, 2 * B + 1, 2, dtype=torch.int32, device="cuda")
    p = torch.softmax(row.double() / 0.8, -1)
    qp = torch.softmax(torch.tensor([0.0, 1.0, 0.5, 0.3, -1.0, 0.0], device="cuda"), -1)
    for probs in (False, True):
        gum = -torch.log(torch.empty(B, V, device="cuda").exponential_(generator=g))
        u = torch.rand(2 * B, generator=g, device="cuda")
        if probs:
            drafts = torch.multinomial(qp, 2 * B, replacement=True, generator=g).to(torch.int32)
        else:
            drafts = torch.full((2 * B,), 3, dtype=torch.int32, device="cuda")
        tokens, _, _ = paged.verify_drafts(logits, begin, drafts, u, gum, torch.full((B,), 0.8, device="cuda"), 1,
                                           draft_probs=qp.expand(2 * B, V).contiguous() if probs else None)
        f = torch.bincount(tokens[:, 0].long(), minlength=V).double() / B
        assert ((f - p).abs() <= 5 * (p * (1 - p) / B).sqrt() + 1e-12).all(), (probs, f.tolist(), p.tolist())


# ------------------------------------------------------------------------------ together

@pytest.mark.parametrize("fmt,window", [("int8", 0), ("e4m3", 24), ("bf16", 0)])
def test_example_speculation_gives_the_plain_greedy_tokens(paged, cuda, fmt, window):
    """The example's server: with drafts, in fewer passes, the tokens that one at a time gives."""
    example = importlib.import_module("examples.paged_speculation")
    out = example.main(["--tokens", "40", "--format", fmt, "--window", str(window)])
    assert out["ids"] == out["plain"] and all(len(x) == 40 for x in out["ids"])
    assert out["plain_passes"] == 40 and out["passes"] < 40 and out["accepted"] > 0


def test_example_samples_at_a_temperature(paged, cuda):
    example = importlib.import_module("examples.paged_speculation")
    out = example.main(["--tokens", "12", "--temperature", "0.9"])
    assert all(len(x) == 12 and all(0 <= t < 384 for t in x) for x in out["ids"])


@pytest.mark.parametrize("q_len", [1, 40])
@pytest.mark.parametrize("window", [0, 40])
def test_e4m3_positions_that_no_row_sees_may_hold_nan_codes(paged, cuda, q_len, window):
    """Memory of a page that was never written, or that belongs to positions below the window."""
    torch = cuda
    kv = 150
    table, pages = layout(torch, [kv], 64, 1, 4)
    pool = make_pool(paged, torch, "e4m3", pages, 64, 1, 128, 4)
    pos = kv - q_len
    lo = max(0, pos - window + 1) if window else 0
    for x in (pool.k, pool.v):
        raw = x.view(torch.uint8)
        for t in list(range(0, lo)) + list(range(kv, 3 * 64)):
            raw[int(table[0, t // 64]), :, t % 64] = 0x7F
    q = torch.randn(q_len, 8, 128, generator=gen(torch, 9), device="cuda").bfloat16()
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    out = paged.attention(pool, q, ints([0, q_len]), ints([pos]), ints([kv]), table, q_len, kv, window=window, scale=0.05)
    want = reference(torch, pool, q, [(0, q_len, pos, kv)], table, window, float(np.float32(0.05)))
    check(torch, out, None, *want, True)


@pytest.mark.parametrize("q_len", [2, 40])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_bf16_values_a_row_does_not_see_never_reach_it(paged, cuda, q_len, bad):
    """One new token's V holds a value that is not finite: the rows before it stay finite and right, those
    from it on are not finite where the value enters."""
    torch = cuda
    kv = 100
    table, pages = layout(torch, [kv], 16, 1, 4)
    pool = make_pool(paged, torch, "bf16", pages, 16, 1, 128, 4)
    q = torch.randn(q_len, 8, 128, generator=gen(torch, 9), device="cuda").bfloat16()
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    args = (ints([0, q_len]), ints([kv - q_len]), ints([kv]), table, q_len, kv)
    good = paged.attention(pool, q, *args, scale=0.05)
    pool.v[int(table[0, (kv - 1) // 16]), 0, (kv - 1) % 16, 5] = bad
    out = paged.attention(pool, q, *args, scale=0.05)
    assert torch.equal(out[:-1], good[:-1])
    assert not out[-1, :, 5].isfinite().any()


@pytest.mark.parametrize("fmt,page,q_len", [("bf16", 1024, 1), ("bf16", 1024, 40), ("int8", 1024, 1), ("int8", 1024, 40)])
def test_offsets_past_32_bits(paged, cuda, fmt, page, q_len):
    """The last pages of a pool of more than 2^32 bytes (and 2^31 values) give what the same rows give in
    a small pool, bit for bit."""
    torch = cuda
    heads, hd = 8, 512
    pages = (2 ** 32 // (heads * page * hd * (2 if fmt == "bf16" else 1))) + 3
    big = paged.PagePool.create(pages, page, heads, hd, fmt)
    small = paged.PagePool.create(2, page, heads, hd, fmt)
    kv = page + 300
    k = torch.randn(kv, heads, hd, generator=gen(torch, 1), device="cuda").bfloat16()
    v = torch.randn(kv, heads, hd, generator=gen(torch, 2), device="cuda").bfloat16()
    q = torch.randn(q_len, 2 * heads, hd, generator=gen(torch, 3), device="cuda").bfloat16()
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    outs = []
    for pool, ids in ((big, [pages - 1, pages - 2]), (small, [1, 0])):
        slots = torch.tensor([ids[t // page] * page + t % page for t in range(kv)], dtype=torch.int32, device="cuda")
        pool.store(k, v, slots)
        out = paged.attention(pool, q, ints([0, q_len]), ints([kv - q_len]), ints([kv]), ints([ids]), q_len, kv, scale=0.04)
        outs.append((out, *pool.read(slots, torch.bfloat16)))
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    assert outs[0][0].float().abs().max() > 0 and (outs[0][1].float() - k.float()).abs().max() < 0.05
    del big
    torch.cuda.empty_cache()
