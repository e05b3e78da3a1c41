"""Serving operators over a paged cache on the GPU: each against a plain form in 64 bits at the sizes, layouts and masks where it can go wrong, and a step
of all of them as a program strings them together."""
import math

import pytest
import torch

import serving_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def sv(ofa):
    return ofa.serving


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def starts(new):
    s = [0]
    for n in new:
        s.append(s[-1] + n)
    return s


def make(sv, new, kv, kv_heads, dim, page, dtype="bf16", layout="heads", seed=0, spare=2, **hints):
    """A cache in use: pages anywhere, all its rows filled by kv_append's own rule on the host, and a batch of sequences."""
    g = torch.Generator().manual_seed(seed)
    per = [-(-max(k, 0) // page) for k in kv]
    n_pages = sum(per) + spare
    perm = torch.randperm(n_pages, generator=g).tolist()
    cols = max(per + [1])
    table, at = [], 0
    for n in per:
        table.append(perm[at:at + n] + [-1] * (cols - n))
        at += n
    shape = (n_pages, kv_heads, page) if layout == "heads" else (n_pages, page, kv_heads)
    pools, scales = [], []
    for _ in range(2):
        x = (torch.randn(*shape, dim, generator=g) * torch.exp2(torch.randint(-3, 3, shape, generator=g).float())[..., None]).bfloat16()
        if dtype == "e4m3":
            q, b = ref.quantise(x)
            x = q.float().to(torch.float8_e4m3fn)
            scales.append(b.to(DEV) if layout == "heads" else b.to(DEV).transpose(1, 2))
        x = x.to(DEV)
        pools.append(x if layout == "heads" else x.transpose(1, 2))
    cache = sv.KVCache(*pools, *scales)
    st = starts(new)
    batch = sv.KVBatch(i32(st), i32(kv), i32(table).view(len(kv), cols), status=torch.zeros(1, dtype=torch.int32, device=DEV), **hints)
    return cache, batch, g


def check_attention(sv, cache, batch, q, causal=True, window=0, scale=None):
    got, lse = sv.paged_attention(cache, batch, q, causal=causal, window=window, scale=scale, with_lse=True)
    want, want_lse, tol, tol_lse = ref.attention(cache, batch.q_start.tolist(), batch.kv_len.tolist(), batch.pages.cpu(), q,
                                                 1 / math.sqrt(cache.head_dim) if scale is None else scale, causal, window)
    rows = ~torch.isnan(want_lse[:, 0]) if want_lse.numel() else torch.zeros(0, dtype=torch.bool)
    got, lse = got.double().cpu(), lse.double().cpu()
    off = (got - want).abs()[rows]
    assert torch.isfinite(got[rows]).all()
    assert (off <= tol[rows]).all(), f"worst error is {float((off / tol[rows].clamp(min=1e-300)).max()):.3g} of its bound"
    none = want_lse[rows] == -math.inf
    assert torch.equal(none, lse[rows] == -math.inf)
    off = (lse - want_lse).abs()[rows][~none]
    assert (off <= tol_lse[rows][~none]).all(), f"lse: {float((off / tol_lse[rows][~none]).max()):.3g} of its bound"
    return got, lse


def queries(g, rows, heads, dim):
    x = torch.randn(rows, (heads + 3) * dim, generator=g).bfloat16().to(DEV)
    return x[:, dim:(heads + 1) * dim].view(rows, heads, dim)           # a view of something wider


# ------------------------------------------------------------------------------------------------ append and read
@pytest.mark.parametrize("layout", ["heads", "rows"])
@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
@pytest.mark.parametrize("new,kv,heads,dim,page", [([1], [1], 1, 64, 1), ([1, 0, 3, 1], [5, 9, 3, 129], 12, 64, 16), ([130, 7], [130, 200], 3, 128, 33),
                                                   ([0], [4], 2, 64, 8), ([1] * 70, list(range(1, 71)), 2, 64, 24)])
def test_rows_go_to_their_pages_and_come_back(sv, new, kv, heads, dim, page, dtype, layout):
    cache, batch, g = make(sv, new, kv, heads, dim, page, dtype, layout)
    rows = sum(new)
    before = [t.clone() for t in (cache.k, cache.v)]
    kvs = torch.randn(rows, 2 * heads * dim, generator=g) * torch.exp2(torch.randint(-30, 12, (rows, 1), generator=g).float())
    kvs = kvs.bfloat16().to(DEV)
    k, v = (t.view(rows, heads, dim) for t in kvs.split(heads * dim, 1))
    sv.kv_append(cache, batch, k, v)
    got = sv.kv_read(cache, batch, rows)
    changed = torch.zeros(cache.n_pages, page, dtype=torch.bool)
    at, table = 0, batch.pages.cpu()
    for i, (n, length) in enumerate(zip(new, kv)):
        for p in range(length - n, length):
            pg, r = int(table[i, p // page]), p % page
            changed[pg, r] = True
            for name, x, back in (("k", k, got[0]), ("v", v, got[1])):
                if dtype == "bf16":
                    want = x[at].double().cpu()
                else:
                    q, b = ref.quantise(x[at])
                    want = q * 2.0 ** (b.double() - 127)[:, None]
                    assert torch.equal(getattr(cache, name + "_scale")[pg, :, r].cpu(), b)
                    assert torch.equal(getattr(cache, name)[pg, :, r].double().cpu(), q)
                assert torch.equal(ref.cached(cache, name, pg, r), want)
                assert torch.equal(back[at].double().cpu(), want), "a read rounds nothing"
            at += 1
    for now, was in zip((cache.k, cache.v), before):                    # and nothing else is touched
        same = (now.contiguous().view(torch.uint8) == was.contiguous().view(torch.uint8)).view(cache.n_pages, heads, page, -1).all(-1).all(1).cpu()
        assert same[~changed].all()
    assert int(batch.status) == 0


def test_every_code_and_scale_reads_back_exactly(sv):
    codes = torch.arange(256, dtype=torch.uint8, device=DEV).repeat(128 * 64 // 256)
    for first in (27, 100, 127, 134 - 63 + 0):
        k = codes.view(torch.float8_e4m3fn).view(1, 1, 128, 64).contiguous()
        k = torch.where(torch.isnan(k.float()), torch.zeros_like(k.float()), k.float()).to(torch.float8_e4m3fn)
        b = (first + torch.arange(128, device=DEV) % 64).clamp(max=134).to(torch.uint8).view(1, 1, 128)
        cache = sv.KVCache(k, k.clone(), b, b.clone())
        batch = sv.KVBatch(i32([0, 128]), i32([128]), i32([[0]]))
        got = sv.kv_read(cache, batch, 128)[0].double()[:, 0]
        want = k.double()[0, 0] * torch.tensor([2.0 ** (int(x) - 127) for x in b.flatten()], dtype=torch.float64, device=DEV)[:, None]
        assert torch.equal(got, want)


def test_rows_with_nan_infinity_zeros_and_the_largest_values(sv):
    cache = sv.KVCache.empty(1, 8, 1, 64, "e4m3")
    batch = sv.KVBatch(i32([0, 6]), i32([6]), i32([[0]]))
    x = torch.randn(6, 1, 64).bfloat16()
    x[0, 0, 3] = math.nan
    x[1, 0, 63] = -math.inf
    x[2] = 0
    x[3, 0, 5] = 3.3e38                                                 # above 448 * 2^7: held as 57344
    x[4] = x[4].float().mul(1e-36).bfloat16()                           # far below the smallest scale
    x[5, 0, 0] = 448.0
    x = x.to(DEV)
    sv.kv_append(cache, batch, x, x)
    assert cache.k_scale[0, 0, :6].tolist()[:4] == [255, 255, 27, 134] and int(cache.k_scale[0, 0, 4]) == 27
    k, _ = sv.kv_read(cache, batch, 6)
    k = k.double().cpu()[:, 0]
    assert torch.isnan(k[0]).all() and torch.isnan(k[1]).all() and (k[2] == 0).all() and float(k[3, 5]) == 57344.0
    assert (k[4].abs() <= 2.0 ** -109).all()
    q, b = ref.quantise(x[5])
    assert torch.equal(k[5], (q * 2.0 ** (b.double() - 127)[:, None])[0])


# ------------------------------------------------------------------------------------------------ attention
CASES = [
    # new, kv, heads, kv_heads, dim, page
    ([1], [1], 1, 1, 64, 16),
    ([1], [1000], 12, 12, 64, 16),
    ([1, 1, 1], [31, 32, 33], 4, 2, 128, 8),
    ([1, 0, 1], [300, 50, 7], 8, 1, 64, 33),
    ([3, 1, 17, 2], [3, 600, 40, 2], 12, 12, 64, 24),
    ([5, 5], [257, 90], 32, 8, 128, 64),
    ([16, 1], [16, 513], 24, 8, 64, 1),
    ([33], [100], 3, 1, 128, 16),
    ([70, 129], [70, 300], 4, 4, 64, 16),
    ([200], [333], 6, 2, 128, 128),
]


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{len(c[0])}x{max(c[0])}of{max(c[1])}_h{c[2]}_{c[3]}_d{c[4]}_p{c[5]}")
def test_attention(sv, case, dtype):
    new, kv, heads, kv_heads, dim, page = case
    cache, batch, g = make(sv, new, kv, kv_heads, dim, page, dtype, "rows" if len(new) % 2 else "heads", max_new=max(new), max_kv=max(kv))
    check_attention(sv, cache, batch, queries(g, sum(new), heads, dim))
    assert int(batch.status) == 0


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
@pytest.mark.parametrize("window", [1, 2, 31, 64, 200])
@pytest.mark.parametrize("new", [[1, 1], [9, 40]])
def test_window(sv, new, window, dtype):
    cache, batch, g = make(sv, new, [500, 77], 2, 64, 16, dtype, max_new=max(new))
    check_attention(sv, cache, batch, queries(g, sum(new), 4, 64), window=window)


@pytest.mark.parametrize("new", [[1, 1], [7, 150]])
def test_without_causal_mask_and_with_another_scale(sv, new):
    cache, batch, g = make(sv, new, [40, 333], 2, 128, 32)
    check_attention(sv, cache, batch, queries(g, sum(new), 4, 128), causal=False, scale=0.3)
    check_attention(sv, cache, batch, queries(g, sum(new), 4, 128), scale=-0.05)


@pytest.mark.parametrize("hints", [{}, {"max_new": 1}, {"max_kv": 1}, {"max_new": 1, "max_kv": 1}, {"max_new": 10 ** 6, "max_kv": 10 ** 9}])
def test_hints_change_no_result_beyond_rounding(sv, hints):
    """max_new and max_kv only choose how the work is cut: too small, too large or absent, every row is computed"""
    new, kv = [60, 1, 5], [900, 2000, 5]
    cache, batch, g = make(sv, new, kv, 2, 64, 16, **hints)
    check_attention(sv, cache, batch, queries(g, sum(new), 4, 64))


@pytest.mark.parametrize("new", [[4, 2, 1], [40, 20, 1]])
def test_rows_that_see_nothing(sv, new):
    """A sequence shorter than what it brings has rows before its first position; one of length 0 has only such rows."""
    cache, batch, g = make(sv, new, [2, 0, 1], 2, 64, 16)
    got, lse = check_attention(sv, cache, batch, queries(g, sum(new), 2, 64))
    assert (got[: new[0] - 2] == 0).all() and (lse[: new[0] - 2] == -math.inf).all()


@pytest.mark.parametrize("new,heads", [([1, 1], 2), ([30, 1], 4)])
def test_rows_of_no_sequence_are_left_alone(sv, new, heads):
    cache, batch, g = make(sv, new, [300, 1200], 2, 64, 16)
    rows = sum(new) + 5
    q = queries(g, rows, heads, 64)
    out = torch.full((rows, heads, 64), 7.0, dtype=torch.bfloat16, device=DEV)
    sv.paged_attention(cache, batch, q, out=out)
    assert (out[sum(new):] == 7).all()
    k = torch.full((rows, 2, 64), 9.0, dtype=torch.bfloat16, device=DEV)
    v = k.clone()
    sv.kv_read(cache, batch, k=k, v=v)
    assert (k[sum(new):] == 9).all() and (v[sum(new):] == 9).all() and not (k[:sum(new)] == 9).all()


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
@pytest.mark.parametrize("new,kv,window", [([5], [70], 0), ([1], [70], 20), ([20], [300], 40), ([150], [300], 0), ([150], [300], 33)])
def test_what_a_row_does_not_see_does_not_reach_it(sv, new, kv, window, dtype):
    """NaN and infinities in keys and values that some rows see and others do not, and in the unused rest of the last page"""
    cache, batch, g = make(sv, new, kv, 1, 64, 64, dtype)
    q = queries(g, new[0], 2, 64)
    table = batch.pages.cpu()
    where = lambda p: (int(table[0, p // 64]), 0, p % 64)  # noqa: E731
    n, length = new[0], kv[0]

    def spoil(p, value):
        if dtype == "e4m3":
            cache.k_scale[where(p)] = 255
            cache.v_scale[where(p)] = 255
        else:
            cache.k[where(p)][3] = value
            cache.v[where(p)][5] = value
            cache.v[where(p)][6] = -value
    spoiled = sorted({length - 1, length - n // 2 - 1} | ({max(0, length - n - window + 1 + n // 3), 0} if window else set())) if n > 1 else ([0] if window else [])
    for p in spoiled:
        spoil(p, math.nan if p % 2 else math.inf)
    last = int(table[0, length // 64])                                   # the rest of the last page was never written
    if dtype == "e4m3":
        cache.k_scale[last, 0, length % 64:] = cache.v_scale[last, 0, length % 64:] = 255
    else:
        cache.k[last, 0, length % 64:] = cache.v[last, 0, length % 64:] = math.nan
    got, lse = sv.paged_attention(cache, batch, q, window=window, with_lse=True)
    got, lse = got.double().cpu(), lse.cpu()
    want, _, tol, _ = ref.attention(cache, [0, n], kv, table, q, 1 / 8, True, window)
    clean = torch.tensor([not any(p <= length - n + t and (not window or p > length - n + t - window) for p in spoiled) for t in range(n)])
    assert clean.any()
    assert torch.isfinite(got[clean]).all() and ((got - want).abs()[clean] <= tol[clean]).all()
    if dtype == "e4m3":
        assert torch.isnan(got[~clean]).all() and torch.isnan(lse[~clean]).all()
    assert not torch.isfinite(got[~clean][..., 5]).any()


@pytest.mark.parametrize("new", [[6], [100]])
def test_infinite_values_reach_the_rows_that_see_them(sv, new):
    cache, batch, g = make(sv, new, [160], 1, 64, 32)
    table = batch.pages.cpu()
    p = 160 - new[0] // 2
    pg, r = int(table[0, p // 32]), p % 32
    cache.v[pg, 0, r, 9] = math.inf
    cache.v[pg, 0, r, 40] = math.nan
    q = queries(g, new[0], 2, 64)
    got = sv.paged_attention(cache, batch, q).float().cpu()
    sees = torch.arange(160 - new[0], 160) >= p
    assert (got[sees][:, :, 9] == math.inf).all() and torch.isnan(got[sees][:, :, 40]).all()
    others = [d for d in range(64) if d not in (9, 40)]
    want, _, tol, _ = ref.attention(cache, [0, new[0]], [160], table, q, 1 / 8)
    assert torch.isfinite(got[~sees]).all()
    assert ((got.double() - want).abs()[:, :, others] <= tol[:, :, others]).all()


@pytest.mark.parametrize("new", [[2], [90]])
def test_bad_tables_and_lengths_set_status_and_nothing_else(sv, new):
    n = new[0]
    cache, batch, g = make(sv, new, [200], 2, 64, 16)
    q = queries(g, n, 4, 64)
    batch.pages[0, 3], batch.pages[0, 7] = cache.n_pages, -5              # their keys are not seen
    check_attention(sv, cache, batch, q)
    assert int(batch.status) == sv.BAD_PAGE
    long = sv.KVBatch(i32([0, n]), i32([10 ** 9]), batch.pages, status=torch.zeros(1, dtype=torch.int32, device=DEV))
    sv.paged_attention(cache, long, q, window=1000)
    k, v = sv.kv_read(cache, long, n)
    assert int(long.status) & sv.BAD_LENGTH and (k == 0).all() and (v == 0).all()
    before = cache.k.clone()
    sv.kv_append(cache, long, q[:, :2], q[:, :2])
    assert torch.equal(before, cache.k)
    for st in ([0, n + 1], [-1, n], [n, 0]):
        bad = sv.KVBatch(i32(st), i32([100]), batch.pages, status=torch.zeros(1, dtype=torch.int32, device=DEV))
        out = torch.full((n, 4, 64), 3.0, dtype=torch.bfloat16, device=DEV)
        sv.paged_attention(cache, bad, q, out=out)
        sv.kv_append(cache, bad, q[:, :2], q[:, :2])
        assert int(bad.status) & sv.BAD_ROWS and torch.equal(before, cache.k)
    neg = sv.KVBatch(i32([0, n]), i32([-3]), batch.pages, status=torch.zeros(1, dtype=torch.int32, device=DEV))
    assert (sv.paged_attention(cache, neg, q) == 0).all() and int(neg.status) & sv.BAD_LENGTH


def test_a_long_cache_whose_offsets_pass_32_bits(sv):
    """4.3 GB of keys: pages beyond 2^32 bytes are the ones in use"""
    pages, page, heads, dim = 16500, 128, 8, 128
    k = torch.empty(pages, heads, page, dim, dtype=torch.bfloat16, device=DEV)
    v = torch.empty_like(k)
    cache = sv.KVCache(k, v)
    table = i32([[pages - 1, pages - 3]])
    g = torch.Generator().manual_seed(1)
    rows = torch.randn(200, 2 * heads * dim, generator=g).bfloat16().to(DEV)
    kk, vv = (t.view(200, heads, dim) for t in rows.split(heads * dim, 1))
    full = sv.KVBatch(i32([0, 200]), i32([200]), table)
    sv.kv_append(cache, full, kk, vv)
    back = sv.kv_read(cache, full, 200)
    assert torch.equal(back[0], kk) and torch.equal(back[1], vv)
    for n in (1, 40):
        batch = sv.KVBatch(i32([0, n]), i32([200]), table)
        q = queries(g, n, 16, dim)
        got = sv.paged_attention(cache, batch, q).double().cpu()
        small = sv.KVCache(k[[pages - 1, pages - 3]].clone(), v[[pages - 1, pages - 3]].clone())
        want, _, tol, _ = ref.attention(small, [0, n], [200], torch.tensor([[0, 1]]), q, 1 / math.sqrt(dim))
        assert ((got - want).abs() <= tol).all()


# ------------------------------------------------------------------------------------------------ logits
def logit_inputs(rows, vocab, history, biases, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, vocab, generator=g) * 4).to(dtype)
    x[0, 0] = -math.inf
    if vocab > 3:
        x[0, 3] = torch.finfo(dtype).min
    a = {}
    if history:
        a["tokens"] = torch.randint(-2, vocab + 2, (rows, history), generator=g).int()
        a["tokens"][:, : history // 2] %= max(1, vocab // 7)              # repeats
        a["n_tokens"] = torch.randint(0, history + 3, (rows,), generator=g).int()
        a["n_prompt"] = torch.randint(0, history + 1, (rows,), generator=g).int()
        a["repetition"] = 1 + torch.rand(rows, generator=g)
        a["presence"], a["frequency"] = torch.rand(rows, generator=g), torch.rand(rows, generator=g) - 0.3
    if biases:
        a["bias_ids"] = torch.randint(-2, vocab + 2, (rows, biases), generator=g).int()
        a["bias_ids"][:, -1] = a["bias_ids"][:, 0]                        # the same id twice
        a["bias"] = torch.randn(rows, biases, generator=g) * 5
    return x, a, torch.randint(-2 ** 31, 2 ** 31, (rows, (vocab + 31) // 32), generator=g).int()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,history,biases,masked", [(1, 1, 3, 2, True), (3, 33, 40, 5, True), (2, 4097, 0, 0, True), (5, 8191, 300, 9, False), (1, 50304, 1000, 0, True),
                                                              (4, 1000, 0, 3, False), (2, 777, 50, 0, False), (130, 64, 2, 1, True)])
def test_logits(sv, rows, vocab, history, biases, masked, dtype):
    x, a, mask = logit_inputs(rows, vocab, history, biases, dtype)
    if masked:
        mask[-1] = 0                                                      # a row that may take nothing
        a["mask"] = mask
    want, tol = ref.logits(x, **a)
    half = ref.F32_HALF if dtype == torch.float32 else ref.BF16_HALF
    tol = tol + half * (want.abs() + tol)
    dev = {k: v.to(DEV) for k, v in a.items()}
    got = sv.logits_process(x.to(DEV), **dev)
    place = x.to(DEV)
    assert sv.logits_process(place, out=place, **dev) is place
    assert torch.equal(got, place)
    got, fine = got.double().cpu(), torch.isfinite(want)
    over = want.abs() >= torch.finfo(dtype).max                           # the lowest value times a factor is -inf in the type
    same = fine & ~over
    assert torch.equal(got[~fine], want[~fine])
    assert ((got - want).abs()[same] <= tol[same]).all()
    assert (got[fine & over] == -math.inf).all() or (got[fine & over] == torch.finfo(dtype).min).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,history,biases,masked", [(700, 1000, 50, 6, True), (700, 300, 5000, 0, False), (620, 2000, 8300, 3, True), (170, 33001, 8000, 192, True), (170, 33001, 0, 7, False),
                                                              (170, 33000, 0, 0, True), (9000, 5, 3, 1, True)])
def test_logits_of_many_rows(sv, rows, vocab, history, biases, masked, dtype):
    """bit by bit what a few of the rows give alone; some against the plain form"""
    x, a, mask = logit_inputs(rows, vocab, history, biases, dtype, seed=3)
    if masked:
        a["mask"] = mask
    dev, x = {k: v.to(DEV) for k, v in a.items()}, x.to(DEV)
    got = sv.logits_process(x, **dev)
    for r in range(0, rows, 8 if rows < 1000 else 500):
        part = slice(r, r + 8)
        assert torch.equal(got[part], sv.logits_process(x[part], **{k: v[part] for k, v in dev.items()}))
    some = slice(rows - 3, rows)
    want, tol = ref.logits(x[some], **{k: v[some] for k, v in a.items()})
    tol = tol + (ref.F32_HALF if dtype == torch.float32 else ref.BF16_HALF) * (want.abs() + tol)
    fine, have = torch.isfinite(want), got[some].double().cpu()
    assert torch.equal(have[~fine], want[~fine]) and ((have - want).abs()[fine] <= tol[fine]).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = sv.logits_process(x, **dev)
    again.zero_()
    graph.replay()
    assert torch.equal(again, got)
    assert sv.logits_process(x, out=x, **dev) is x and torch.equal(x, got)


def test_logits_of_strided_rows(sv):
    wide = torch.randn(4, 3000, device=DEV)
    x = wide[:, 5:1006]
    mask = torch.randint(-2 ** 31, 2 ** 31, (4, 40), device=DEV).int()[:, 3:35]
    bias_ids, bias = torch.randint(0, 1001, (4, 6), device=DEV).int()[:, :4], torch.randn(4, 6, device=DEV)[:, :4]
    want, tol = ref.logits(x, bias_ids=bias_ids.cpu(), bias=bias.cpu(), mask=mask)
    before = wide.clone()
    got = sv.logits_process(x, bias_ids=bias_ids, bias=bias, mask=mask)
    assert torch.equal(wide, before)
    fine = torch.isfinite(want)
    assert torch.equal(got.cpu()[~fine].double(), want[~fine]) and ((got.cpu().double() - want).abs()[fine] <= (tol + want.abs() * ref.F32_HALF)[fine]).all()
    sv.logits_process(x, bias_ids=bias_ids, bias=bias, mask=mask, out=x)
    assert torch.equal(x, got) and torch.equal(wide[:, :5], before[:, :5]) and torch.equal(wide[:, 1006:], before[:, 1006:])


# ------------------------------------------------------------------------------------------------ together
def plain_step(sv, cache, lens, table, qkv, heads, kv_heads, dim):
    n = [1] * len(lens)
    return ref.attention(cache, starts(n), lens, table, qkv[:, : heads * dim].view(len(lens), heads, dim), 1 / math.sqrt(dim))


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
def test_a_serving_run(sv, dtype):
    """Prompts in one chunk, then tokens one at a time: append, attend, logits; the steps are also captured once and replayed with the lengths, tokens
    and rows of each step, on another stream than the default one, and give the same bits."""
    heads, kv_heads, dim, page, vocab, steps = 4, 2, 64, 16, 500, 5
    prompt = [40, 3, 17]
    kv = [p + steps for p in prompt]
    cache, batch, g = make(sv, prompt, kv, kv_heads, dim, page, dtype)
    width = (heads + 2 * kv_heads) * dim
    head = torch.randn(heads * dim, vocab, generator=g).to(DEV) * 0.1

    def step(c, b, x):
        q, k, v = (t.view(x.shape[0], -1, dim) for t in x.split([heads * dim, kv_heads * dim, kv_heads * dim], 1))
        sv.kv_append(c, b, k, v)
        return sv.paged_attention(c, b, q)
    chunk = torch.randn(sum(prompt), width, generator=g).bfloat16().to(DEV)
    first = sv.KVBatch(i32(starts(prompt)), i32(prompt), batch.pages, max_new=40)
    o = step(cache, first, chunk)
    want, _, tol, _ = ref.attention(cache, starts(prompt), prompt, batch.pages.cpu(), chunk[:, : heads * dim].view(-1, heads, dim), 1 / 8)
    assert ((o.double().cpu() - want).abs() <= tol).all()

    xs = [torch.randn(3, width, generator=g).bfloat16().to(DEV) for _ in range(steps)]
    history = torch.zeros(3, steps, dtype=torch.int32, device=DEV)
    pen = {"repetition": torch.full((3,), 1.3, device=DEV), "frequency": torch.full((3,), 0.2, device=DEV)}

    def run(c, step_batch, lens, x, hist, made):
        o = step(c, step_batch, x)
        return o, sv.logits_process((o.reshape(3, -1).float() @ head), tokens=hist, n_tokens=made, **pen)
    snapshot = [t.clone() for t in (cache.k, cache.v)] + ([cache.k_scale.clone(), cache.v_scale.clone()] if dtype == "e4m3" else [])
    eager = []
    for s in range(steps):
        lens = [p + s + 1 for p in prompt]
        b = sv.KVBatch(i32([0, 1, 2, 3]), i32(lens), batch.pages, max_new=1, max_kv=max(kv))
        o, y = run(cache, b, lens, xs[s], history, i32([s] * 3))
        want, _, tol, _ = plain_step(sv, cache, lens, batch.pages.cpu(), xs[s], heads, kv_heads, dim)
        assert ((o.double().cpu() - want).abs() <= tol).all()
        want, tol = ref.logits((o.reshape(3, -1).float() @ head), tokens=history.cpu(), n_tokens=[s] * 3, **{k: v.cpu() for k, v in pen.items()})
        assert ((y.double().cpu() - want).abs() <= tol + want.abs() * ref.F32_HALF).all()
        history[:, s] = y.argmax(-1).int()
        eager.append((o.clone(), y.clone()))
    for t, was in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), snapshot):
        t.copy_(was)
    made, length, x = i32([0] * 3), i32([p + 1 for p in prompt]), xs[0].clone()
    hist = torch.zeros_like(history)
    b = sv.KVBatch(i32([0, 1, 2, 3]), length, batch.pages, max_new=1, max_kv=max(kv))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        o, y = run(cache, b, None, x, hist, made)
    for s in range(steps):
        x.copy_(xs[s])
        made.fill_(s)
        length.copy_(i32([p + s + 1 for p in prompt]))
        graph.replay()
        assert torch.equal(o, eager[s][0]) and torch.equal(y, eager[s][1])
        hist[:, s] = y.argmax(-1).int()


def test_calls_on_two_streams_at_once(sv):
    """Each with its own workspace: the same bits as one after the other"""
    a = make(sv, [1, 1], [3000, 900], 2, 64, 16, seed=1)
    b = make(sv, [3], [4000], 2, 64, 16, "e4m3", seed=2)
    qa, qb = queries(a[2], 2, 8, 64), queries(b[2], 3, 8, 64)
    want = sv.paged_attention(a[0], a[1], qa).clone(), sv.paged_attention(b[0], b[1], qb).clone()
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(20):
        with torch.cuda.stream(s1):
            x = sv.paged_attention(a[0], a[1], qa)
        with torch.cuda.stream(s2):
            y = sv.paged_attention(b[0], b[1], qb)
        got.append((x, y))
    torch.cuda.synchronize()
    for x, y in got:
        assert torch.equal(x, want[0]) and torch.equal(y, want[1])


def test_empty_calls(sv):
    cache, batch, _ = make(sv, [0, 0], [5, 0], 2, 64, 16)
    e = torch.empty(0, 2, 64, dtype=torch.bfloat16, device=DEV)
    sv.kv_append(cache, batch, e, e)
    assert sv.kv_read(cache, batch, 0)[0].shape == (0, 2, 64)
    assert sv.paged_attention(cache, batch, e).shape == (0, 2, 64)
    none = sv.KVBatch(i32([0]), torch.empty(0, dtype=torch.int32, device=DEV), torch.empty(0, 4, dtype=torch.int32, device=DEV))
    assert sv.paged_attention(cache, none, e).shape == (0, 2, 64)
    assert sv.logits_process(torch.empty(0, 10, device=DEV)).shape == (0, 10)


@pytest.mark.parametrize("rows", [1, 5, 40])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_over_codes_of_every_size(sv, dim, rows):
    """8-bit rows of subnormal codes, of the smallest and largest scales, and queries of any magnitude: nothing underflows or overflows on the way. Scales of keys and
    queries are opposite, so that scores are of order one."""
    g = torch.Generator().manual_seed(3)
    n = 96
    codes = torch.randint(0, 256, (2, n, dim), generator=g).to(torch.uint8)
    codes[:, : n // 3] &= 0x87                                            # subnormal
    codes[(codes & 0x7f) == 0x7f] = 0x7e
    for e in (-100, -60, 0, 7):
        k = codes[0].view(torch.float8_e4m3fn).view(1, 1, n, dim).to(DEV)
        v = codes[1].view(torch.float8_e4m3fn).view(1, 1, n, dim).to(DEV)
        ks = torch.full((1, 1, n), e + 127, dtype=torch.uint8, device=DEV)
        vs = torch.randint(27, 135, (1, 1, n), generator=g).to(torch.uint8).to(DEV) if e == 0 else ks.clone()
        cache = sv.KVCache(k, v, ks, vs)
        batch = sv.KVBatch(i32([0, rows]), i32([n]), i32([[0]]), max_new=rows)
        q = (torch.randn(rows, 2, dim, generator=g) * 2.0 ** (-e - 8)).bfloat16().to(DEV)
        check_attention(sv, cache, batch, q)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,pad", [(3, 8200, 1), (600, 4103, 0), (9, 2049, 3), (2, 7, 5), (200, 12289, 2)])
def test_logits_of_rows_between_boundaries(sv, rows, vocab, pad, dtype):
    """Odd vocabularies and offsets: rows start anywhere against 16 bytes, in one tensor alike and in the other not"""
    x, a, mask = logit_inputs(rows, vocab, 20, 3, dtype)
    a["mask"] = mask
    dev = {k: v.to(DEV) for k, v in a.items()}
    half = ref.F32_HALF if dtype == torch.float32 else ref.BF16_HALF
    some = sorted({0, 1, rows // 2, rows - 1})
    want, tol = ref.logits(x[some], **{k: v[some] for k, v in a.items()})
    for shift in (0, pad):
        space = torch.zeros(rows * (vocab + pad) + 8, dtype=dtype, device=DEV)
        y = space[shift: shift + rows * (vocab + pad)].view(rows, vocab + pad)[:, :vocab]
        y.copy_(x.to(DEV))
        for out in (None, torch.empty_like(x.to(DEV)), y):
            got = sv.logits_process(y, out=out, **dev)[some].double().cpu()
            fine = torch.isfinite(want) & (want.abs() < torch.finfo(dtype).max)
            assert torch.equal(got[want == -math.inf], want[want == -math.inf])
            assert ((got - want).abs()[fine] <= (tol + half * (want.abs() + tol))[fine]).all()


@pytest.mark.parametrize("new", [1, 3, 40])
@pytest.mark.parametrize("page", [16, 8, 33])
def test_a_cache_full_of_nan_behind_the_contexts(sv, page, new):
    """Pages that were never written, or held another sequence, may hold anything: contexts end in the middle of boxes, tiles and pages."""
    for length in (new, 45, 130, 256, 300):
        if length < new:
            continue
        cols = -(-length // page)
        cache = sv.KVCache(torch.full((cols, 2, page, 64), math.nan, dtype=torch.bfloat16, device=DEV), torch.full((cols, 2, page, 64), -math.inf, dtype=torch.bfloat16, device=DEV))
        g = torch.Generator().manual_seed(length)
        table = i32([torch.randperm(cols, generator=g).tolist()])
        rows = torch.randn(length, 2, 64, generator=g).bfloat16().to(DEV)
        sv.kv_append(cache, sv.KVBatch(i32([0, length]), i32([length]), table), rows, rows * 2)
        check_attention(sv, cache, sv.KVBatch(i32([0, new]), i32([length]), table, max_new=new), queries(g, new, 4, 64))


def test_thousands_of_sequences(sv):
    """Every block finds its rows among all sequences"""
    n = 3000
    g = torch.Generator().manual_seed(5)
    new = torch.randint(0, 3, (n,), generator=g).tolist()
    kv = [k + int(x) for k, x in zip(new, torch.randint(0, 30, (n,), generator=g))]
    per = [-(-k // 8) for k in kv]
    cols, total = max(per), sum(per)
    perm, at, table = torch.randperm(total, generator=g).tolist(), 0, []
    for p in per:
        table.append(perm[at:at + p] + [-1] * (cols - p))
        at += p
    cache = sv.KVCache.empty(total, 8, 1, 64)
    full = sv.KVBatch(i32(starts(kv)), i32(kv), i32(table))
    k, v = (torch.randn(sum(kv), 1, 64, generator=g).bfloat16().to(DEV) for _ in range(2))
    sv.kv_append(cache, full, k, v)
    back = sv.kv_read(cache, full, sum(kv))
    assert torch.equal(back[0], k) and torch.equal(back[1], v)
    q = queries(g, sum(new), 2, 64)
    o, lse = sv.paged_attention(cache, sv.KVBatch(i32(starts(new)), i32(kv), i32(table), max_new=2), q, with_lse=True)
    st = starts(new)
    some = [i for i in range(n) if new[i]][::97]
    for i in some:
        s, e = starts(kv[:i + 1])[-2:]
        want, _, tol, _ = dense(q[st[i]:st[i + 1]], k[s:e], v[s:e])
        assert ((o[st[i]:st[i + 1]].double().cpu() - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
@pytest.mark.parametrize("n", [128, 129])
def test_sequences_by_length(sv, n, dtype):
    """enough of them that blocks start one after the other; equal and missing lengths among them"""
    g = torch.Generator().manual_seed(n)
    kv = [int(x) for x in torch.randint(1, 500, (n,), generator=g)]
    kv[3] = kv[7] = kv[90] = 499
    new = [1] * n
    new[5], kv[5], new[6] = 0, 0, 0
    cache, batch, g = make(sv, new, kv, 4, 64, 16, dtype, max_new=1, max_kv=500)
    check_attention(sv, cache, batch, queries(g, sum(new), 4, 64))


def dense(q, k, v):
    """attention of one sequence whose keys and values lie side by side"""
    class One:
        n_pages, page_size, n_kv_heads, head_dim, k_scale = 1, k.shape[0], k.shape[1], k.shape[2], None
    One.k, One.v = k.transpose(0, 1)[None], v.transpose(0, 1)[None]
    return ref.attention(One, [0, q.shape[0]], [k.shape[0]], torch.tensor([[0]]), q, 1 / math.sqrt(k.shape[2]))


def test_calls_without_the_extension_give_the_same(sv, monkeypatch):
    cache, batch, g = make(sv, [3, 30], [70, 90], 2, 64, 16, "e4m3", max_new=30)
    q = queries(g, 33, 4, 64)
    rows = torch.randn(33, 2, 64, generator=g).bfloat16().to(DEV)
    x, a, mask = logit_inputs(5, 300, 20, 3, torch.float32)
    a = {k: v.to(DEV) for k, v in a.items()} | {"mask": mask.to(DEV)}

    def all_of_them():
        sv.kv_append(cache, batch, rows, rows)
        return (*sv.kv_read(cache, batch, 33), *sv.paged_attention(cache, batch, q, window=50, with_lse=True), sv.logits_process(x.to(DEV), **a))
    assert sv._fast() is not None
    one = all_of_them()
    monkeypatch.setattr(sv, "_fast_module", None)
    for u, w in zip(one, all_of_them()):
        assert torch.equal(u, w)


@pytest.mark.parametrize("extension", [True, False])
def test_tensors_that_do_not_fit_are_refused(sv, ofa, monkeypatch, extension):
    """and nothing is written"""
    if not extension:
        monkeypatch.setattr(sv, "_fast_module", None)
    cache, batch, g = make(sv, [2, 1], [20, 9], 2, 64, 16)
    q, k = queries(g, 3, 4, 64), torch.randn(3, 2, 64, generator=g).bfloat16().to(DEV)
    before = cache.k.clone(), cache.v.clone()
    wide = torch.randn(3, 2, 128, device=DEV).bfloat16()
    for bad in (k.float(), k.half(), k[:, :1], k[..., :32], wide[..., ::2], k.cpu(), k[0], None, "k", k.transpose(0, 1)):
        with pytest.raises(ofa.OfaError):
            sv.kv_append(cache, batch, bad, k)
        with pytest.raises(ofa.OfaError):
            sv.kv_append(cache, batch, k, bad)
    for bad in (q.float(), q[..., :32], torch.randn(3, 4, 128, device=DEV).bfloat16()[..., ::2], q.cpu(), q[0], None, q[:, :3], torch.randn(3, 4, 65, device=DEV).bfloat16()[..., 1:]):
        with pytest.raises(ofa.OfaError):
            sv.paged_attention(cache, batch, bad)
    for more in ({"window": -1}, {"window": 3, "causal": False}, {"scale": math.nan}, {"out": q.float()}, {"out": torch.empty_like(q)[:2]}, {"out": torch.empty_like(q)[:1].expand(3, -1, -1)}):
        with pytest.raises(ofa.OfaError):
            sv.paged_attention(cache, batch, q, **more)
    with pytest.raises(ofa.OfaError):
        sv.kv_read(cache, batch)
    with pytest.raises(ofa.OfaError):
        sv.kv_read(cache, batch, 3, k=k)
    with pytest.raises(ofa.OfaError):
        sv.kv_read(cache, batch, 3, k=k, v=k.float())
    x, n = torch.randn(3, 100, device=DEV), i32([1, 2, 3])
    t, f = i32([[1, 2], [3, 4], [5, 6]]), torch.ones(3, device=DEV)
    for more in ({"n_tokens": n}, {"repetition": f}, {"tokens": t.long()}, {"tokens": t, "n_tokens": n.long()}, {"tokens": t[:2]}, {"tokens": t, "repetition": f.double()}, {"tokens": t, "presence": f[:2]},
                 {"bias_ids": t}, {"bias": torch.ones(3, 2, device=DEV)}, {"bias_ids": t, "bias": torch.ones(3, 3, device=DEV)}, {"mask": i32([[1] * 3] * 3)}, {"mask": i32([[1] * 4] * 2)},
                 {"out": x.bfloat16()}, {"out": x[:2]}, {"out": x.t()}, {"tokens": t.t().contiguous().t()}, {"mask": torch.zeros(3, 4, dtype=torch.int32)}, {"out": x[:1].expand(3, -1)}):
        with pytest.raises(ofa.OfaError):
            sv.logits_process(x, **more)
    for bad in (x.half(), x[0], x.cpu(), x.t(), x[:, ::2]):
        with pytest.raises(ofa.OfaError):
            sv.logits_process(bad)
    assert torch.equal(before[0], cache.k) and torch.equal(before[1], cache.v)
    kk, vv = cache.k, cache.v
    for args in ((kk, vv.transpose(1, 2).contiguous().transpose(1, 2)), (kk, vv[:, :1]), (kk, vv.float()), (kk[..., :32], vv[..., :32]), (kk, vv, n, n), (kk.to(torch.float8_e4m3fn), vv.to(torch.float8_e4m3fn)),
                 (torch.zeros(2, 1, 16, 96, dtype=torch.bfloat16, device=DEV),) * 2):
        with pytest.raises(ofa.OfaError):
            sv.KVCache(*args)
    for args in ((n, n, t), (i32([0, 1, 2, 3]).long(), n, t), (i32([0, 1, 2, 3]), n, t.long()), (i32([0, 1, 2, 3]), n.cpu(), t)):
        with pytest.raises(ofa.OfaError):
            sv.KVBatch(*args)
    with pytest.raises(ofa.OfaError):
        sv.KVBatch(i32([0, 1, 2, 3]), n, t, status=torch.zeros(0, dtype=torch.int32, device=DEV))
    with pytest.raises(ofa.OfaError):
        sv.KVBatch(i32([0, 1, 2, 3]), n, t, max_new=-1)


@pytest.mark.parametrize("new,kv", [([1], [400]), ([1] * 70, [300] * 70), ([3, 1], [40, 900]), ([60], [90]), ([130, 3], [3000, 3])])
def test_attention_in_the_place_of_its_queries(sv, new, kv):
    """blocks that share a tile's keys, tiles walked one after the other (a hint that is too small), both kernels"""
    for hints in ({}, {"max_new": 1, "max_kv": max(kv)}):
        cache, batch, g = make(sv, new, kv, 2, 64, 16, **hints)
        q = queries(g, sum(new), 8, 64)
        want = sv.paged_attention(cache, batch, q)
        assert sv.paged_attention(cache, batch, q, out=q) is q and torch.equal(q, want)


def test_logits_side_by_side_in_one_tensor(sv):
    x, a, mask = logit_inputs(6, 333, 30, 4, torch.float32)
    a = {k: v.to(DEV) for k, v in a.items()} | {"mask": mask.to(DEV)}
    both = torch.zeros(6, 700, device=DEV)
    both[:, :333] = x.to(DEV)
    want = sv.logits_process(both[:, :333], **a)
    sv.logits_process(both[:, :333], **a, out=both[:, 367:])
    assert torch.equal(both[:, 367:], want) and torch.equal(both[:, :333], x.to(DEV)) and not both[:, 333:367].any()
    sv.logits_process(both[:, :333], **a, out=both[:, :333])
    assert torch.equal(both[:, :333], want)


def test_two_graphs_share_nothing(sv):
    """each keeps its own workspace; replayed in turns and on two streams at once, after the eager tensors are gone"""
    jobs = []
    for seed, new, kv in ((1, [1, 1], [3000, 2500]), (2, [1, 1, 1], [4000, 100, 2000])):
        cache, batch, g = make(sv, new, kv, 1, 128, 16, seed=seed, max_new=1)
        q = queries(g, sum(new), 4, 128)
        want = sv.paged_attention(cache, batch, q)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = sv.paged_attention(cache, batch, q)
        jobs.append((graph, out, want, s, (cache, batch, q)))
    torch.cuda.synchronize()
    junk = [torch.full((1 << 20,), math.nan, device=DEV) for _ in range(8)]
    for _ in range(5):
        for graph, out, *_ in jobs:
            out.zero_()
        torch.cuda.synchronize()
        for graph, out, want, s, _ in jobs:
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for graph, out, want, *_ in jobs:
            assert torch.equal(out, want)
        for graph, out, want, *_ in jobs:
            graph.replay()
            assert torch.equal(out, want)
    del junk


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [8, 24, 32, 64, 128, 192])
def test_pages_of_many_sizes(sv, page, dim, dtype):
    """boxes of 8 to 64 rows, contexts and windows that begin and end inside them"""
    for new, kv, window in (([1, 1, 1], [1, 63, 300], 0), ([1, 1], [200, 129], 70), ([3, 2], [65, 190], 0), ([40, 9], [40, 333], 0), ([40, 70], [260, 139], 50)):
        cache, batch, g = make(sv, new, kv, 2, dim, page, dtype)
        check_attention(sv, cache, batch, queries(g, sum(new), 8, dim), window=window)


@pytest.mark.parametrize("page", [16, 64, 33])
@pytest.mark.parametrize("new", [1, 40])
def test_a_missing_page_among_others(sv, page, new):
    """its keys are not seen, whatever the box size; the others are"""
    for dtype in ("bf16", "e4m3"):
        cache, batch, g = make(sv, [new], [400], 2, 64, page, dtype)
        bad = batch.pages.clone()
        bad[0, 2] = cache.n_pages + 5
        status = i32([0])
        b2 = sv.KVBatch(batch.q_start, batch.kv_len, bad, status=status)
        q = queries(g, new, 4, 64)
        got, lse = sv.paged_attention(cache, b2, q, with_lse=True)
        assert int(status) == sv.BAD_PAGE
        want, wl, tol, ltol = ref.attention(cache, [0, new], [400], bad.cpu(), q, cache.scale)
        assert ((got.double().cpu() - want).abs() <= tol).all() and ((lse.double().cpu() - wl).abs() <= ltol).all()


@pytest.mark.parametrize("dim,heads", [(128, 8), (64, 8), (128, 2)])
@pytest.mark.parametrize("hint", [3, 5, 12, 30])
def test_chunks_longer_than_the_hint(sv, dim, heads, hint):
    """every form of the kernels walks on through the tiles that the hint did not count"""
    for dtype in ("bf16", "e4m3"):
        cache, batch, g = make(sv, [200, 7, 70], [300, 7, 500], 2, dim, 16, dtype, max_new=hint, max_kv=40)
        check_attention(sv, cache, batch, queries(g, 277, heads, dim))
