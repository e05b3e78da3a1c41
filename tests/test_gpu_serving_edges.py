"""Serving operators on the GPU where calls leave the ordinary: rows that no sequence brings beside split keys, scores without a finite one, the widest windows and longest contexts, queries of
any range, long lists of biases."""
import ctypes as C
import math

import pytest
import torch

import serving_reference as ref
from test_gpu_serving import DEV, check_attention, i32, make, queries, sv  # noqa: F401

pytestmark = pytest.mark.gpu

# Forms of the attention kernels by new tokens and context of a sequence, with two query heads on one key/value head: one block, a cluster of blocks, parts that a second launch joins; few
# rows and many
FORMS = {"few": (2, 20), "few_cluster": (1, 1000), "few_parts": (2, 6000), "many": (40, 90), "many_parts": (40, 6000)}


def call(sv, ofa, cache, batch, q, out, lse, fill=7.0, **more):  # noqa: F811
    """ofa_paged_attention with a workspace that holds something; its size in bytes"""
    lib, K = ofa.capi.load(), ofa.capi
    n, heads, dim = q.shape
    need = lib.ofa_paged_attention_workspace(cache.ref, batch.ref, n, heads)
    work = torch.full((need // 4 + 4,), fill, device=DEV)
    a = K.PagedAttentionArgs(n, heads, q.data_ptr(), q.stride(0), q.stride(1), out.data_ptr(), out.stride(0), out.stride(1), lse.data_ptr(), cache.scale, True, 0, work.data_ptr(), need)
    for k, v in more.items():
        setattr(a, k, v)
    assert lib.ofa_paged_attention(cache.ref, batch.ref, C.byref(a), torch.cuda.current_stream().cuda_stream) == K.OK
    return need


@pytest.mark.parametrize("status", [True, False])
@pytest.mark.parametrize("form", ["few_cluster", "few_parts", "many", "many_parts"])
@pytest.mark.parametrize("kind", ["beyond", "falling", "negative", "alone_beyond", "behind_the_first"])
def test_rows_of_sequences_that_are_left_out_stay_as_they_were(sv, ofa, kind, form, status):  # noqa: F811
    g, kv = FORMS[form]
    n = g + 6
    st, first = {"beyond": ([0, g, n + 90], 0), "falling": ([0, g, g - 1], 0), "negative": ([-1, g], None), "alone_beyond": ([0, n + 1], None), "behind_the_first": ([3, 3 + g], 3)}[kind]
    cache, made, gen = make(sv, [g], [kv], 1, 64, 16)
    seqs = len(st) - 1
    word = i32([0])
    batch = sv.KVBatch(i32(st), i32([kv] * seqs), made.pages.expand(seqs, -1), max_new=g, max_kv=kv, status=word if status else None)
    q = queries(gen, n, 2, 64)
    out, lse = torch.full((n, 2, 64), 3.0, dtype=torch.bfloat16, device=DEV), torch.full((n, 2), 3.0, device=DEV)
    assert (call(sv, ofa, cache, batch, q, out, lse) > 0) == form.endswith("parts")
    have = torch.zeros(n, dtype=torch.bool)
    if first is not None:
        have[first:first + g] = True
        want, want_lse, tol, tol_lse = ref.attention(cache, [first, first + g], [kv], made.pages.cpu(), q, cache.scale)
        assert ((out.double().cpu() - want).abs() <= tol)[have].all() and ((lse.double().cpu() - want_lse).abs() <= tol_lse)[have].all()
    assert (out.cpu()[~have] == 3).all() and (lse.cpu()[~have] == 3).all()
    if status:
        assert int(word) == (0 if kind == "behind_the_first" else sv.BAD_ROWS)


def infinite_query(dtype, form, sv):  # noqa: F811
    """A cache whose keys are all below zero in their first dim, queries of which one, (0, 0), is infinite there"""
    n, kv = FORMS[form]
    cache, batch, gen = make(sv, [n], [kv], 1, 64, 16, dtype, max_new=n, max_kv=kv)
    if dtype == "e4m3":
        cache.k.view(torch.uint8)[..., 0] = 0xb8                         # -1
    else:
        cache.k[..., 0] = -1
    q = queries(gen, n, 2, 64)
    q[0, 0, 0] = math.inf
    return cache, batch, q, n, kv


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
@pytest.mark.parametrize("form", FORMS)
def test_scores_without_a_finite_one(sv, form, dtype):  # noqa: F811
    """exp(x - max x) has no value where every score that a row sees is -inf; a row that sees no key is another matter"""
    cache, batch, q, n, kv = infinite_query(dtype, form, sv)
    out, lse = sv.paged_attention(cache, batch, q, with_lse=True)
    out, lse = out.double().cpu(), lse.double().cpu()
    assert torch.isnan(out[0, 0]).all()
    clean = q.clone()
    clean[0, 0, 0] = 0
    want, want_lse, tol, tol_lse = ref.attention(cache, [0, n], [kv], batch.pages.cpu(), clean, cache.scale)
    some = torch.ones(n, 2, dtype=torch.bool)
    some[0, 0] = False
    assert ((out - want).abs() <= tol)[some].all() and ((lse - want_lse).abs() <= tol_lse)[some].all()
    if dtype == "bf16" or n > 16:
        assert lse[0, 0] == -math.inf
    none = sv.KVBatch(batch.q_start, batch.kv_len, torch.full_like(batch.pages, -1), max_new=n, max_kv=kv)
    for b in (none, sv.KVBatch(batch.q_start, i32([n - 1]), batch.pages, max_new=n, max_kv=kv)):     # no page; one position less than rows
        out, lse = sv.paged_attention(cache, b, q, with_lse=True)
        assert (out[0] == 0).all() and (lse[0] == -math.inf).all()


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 7, 2 ** 31 - 128, 2 ** 30])
@pytest.mark.parametrize("new,kv", [(8, 2), (8, 200), (150, 3), (150, 140), (40, 6000), (4, 6000)])
def test_a_window_wider_than_any_context(sv, new, kv, window, dtype):  # noqa: F811
    """sees what no window sees, in sequences shorter than what they bring too"""
    cache, batch, gen = make(sv, [new], [kv], 1, 64, 16, dtype, max_new=new)
    q = queries(gen, new, 2, 64)
    got, lse = check_attention(sv, cache, batch, q, window=window)
    want, want_lse = sv.paged_attention(cache, batch, q, with_lse=True)
    assert torch.equal(got, want.double().cpu()) and torch.equal(lse, want_lse.double().cpu())


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
@pytest.mark.parametrize("page", [1 << 16, 100003])
@pytest.mark.parametrize("new", [1, 40])
def test_a_context_as_long_as_an_int(sv, new, page, dtype):  # noqa: F811
    """One page that stands throughout a table of 2^31 positions; the last of them, behind 2^31 - 1024, are beyond what a context may have"""
    top, length, window = 2 ** 31 - 1024, 2 ** 31 - 1, 3000
    gen = torch.Generator().manual_seed(page + new)
    cols = -(-2 ** 31 // page)
    table = torch.zeros(1, cols, dtype=torch.int32, device=DEV)
    shape = (1, 1, page, 64)
    if dtype == "e4m3":
        cache = sv.KVCache(*(torch.randn(shape, generator=gen).to(torch.float8_e4m3fn).to(DEV) for _ in range(2)), *(torch.full(shape[:3], 127, dtype=torch.uint8, device=DEV) for _ in range(2)))
    else:
        cache = sv.KVCache(*(torch.randn(shape, generator=gen).bfloat16().to(DEV) for _ in range(2)))
    q = queries(gen, new, 2, 64)
    for kv, status in ((top, 0), (length, sv.BAD_LENGTH)):
        batch = sv.KVBatch(i32([0, new]), i32([kv]), table, max_new=new, max_kv=window, status=i32([0]))
        got, lse = sv.paged_attention(cache, batch, q, window=window, with_lse=True)
        assert int(batch.status) == status
        k, v = (x[0, 0].double().cpu() for x in (cache.k, cache.v))
        for t in range(0, new, 13):
            pos = kv - new + t
            at = torch.arange(pos - window + 1, min(pos + 1, top)) % page
            for h in range(2):
                want, want_lse, tol, tol_lse = one_row(q[t, h].double().cpu(), k[at], v[at], 1 / 8)
                assert ((got[t, h].double().cpu() - want).abs() <= tol).all() and abs(float(lse[t, h]) - want_lse) <= tol_lse


def one_row(q, k, v, scale):
    """(out, lse, their bounds) of one row that sees all of k and v, as serving_reference counts them"""
    x = k @ q * scale
    z = torch.logsumexp(x, 0)
    p = torch.exp(x - z)
    off = float((k.abs() @ q.abs()).max()) * abs(scale) * (len(q) + 16) * 2.0 ** -23 + 2.0 ** -20
    out = p @ v
    return out, float(z), p @ v.abs() * (ref.BF16_HALF + 2 * off) + out.abs() * ref.BF16_HALF * (1 + ref.BF16_HALF) + 1e-37, off + abs(float(z)) * 2.0 ** -22


def held_cache(sv, codes, exponents):  # noqa: F811
    """An 8-bit cache of one page: keys and values of these codes (as floats) [n, dim] and scales 2^e [n]"""
    n, dim = codes[0].shape
    pools = [c.to(torch.float8_e4m3fn).view(1, 1, n, dim).to(DEV) for c in codes]
    return sv.KVCache(*pools, *((e + 127).to(torch.uint8).view(1, 1, n).to(DEV) for e in exponents))


@pytest.mark.parametrize("rows", [1, 3, 5, 8, 16, 40])
@pytest.mark.parametrize("dim", [64, 128])
def test_queries_of_a_wide_range_over_8_bit_keys(sv, dim, rows):  # noqa: F811
    """Scores come from elements far below a row's largest, whose keys are zero: 2^30 below, 2^100 below, and spread over all of it"""
    gen = torch.Generator().manual_seed(dim + rows)
    n = 70
    for low, high, e in ((-6, 24, 7), (-6, 100, 7), (-100, -70, 7), (-6, None, 0)):
        k = torch.randn(n, dim, generator=gen)
        big = torch.arange(dim) % 16 == 5
        if high is not None:
            k[:, big] = 0
        cache = held_cache(sv, [k, torch.randn(n, dim, generator=gen)], [torch.full((n,), float(e)), torch.zeros(n)])
        q = torch.randn(rows, 2, dim, generator=gen) * 2.0 ** low
        if high is None:
            q = q * torch.exp2(torch.randint(-18, 9, (rows, 2, dim), generator=gen).float())
        else:
            q[..., big] = 2.0 ** high * (1 + torch.rand(rows, 2, int(big.sum()), generator=gen))
        q = q.bfloat16().to(DEV)
        batch = sv.KVBatch(i32([0, rows]), i32([n]), i32([[0]]), max_new=rows)
        check_attention(sv, cache, batch, q, scale=0.125 if low > -20 else 2.0 ** 90)


def large_scores(sv, rows, exponent):  # noqa: F811
    """Queries of 2^120 to 2^127 over 8-bit keys of this scale: the row's result is the value of the key whose score is largest by far, its lse that score"""
    gen = torch.Generator().manual_seed(rows)
    n, dim = 50, 64
    k = torch.zeros(n, dim)
    k[:, 3], k[20, 3] = 416.0, 448.0
    v = torch.randn(n, dim, generator=gen)
    cache = held_cache(sv, [k, v], [torch.full((n,), float(exponent)), torch.zeros(n)])
    q = torch.zeros(rows, 1, dim)
    q[:, 0, 3] = 2.0 ** torch.arange(120, 128).float().repeat(-(-rows // 8))[:rows]
    q = q.bfloat16().to(DEV)
    out, lse = sv.paged_attention(cache, sv.KVBatch(i32([0, rows]), i32([n]), i32([[0]]), max_new=rows), q, causal=False, with_lse=True)
    assert (out[:, 0].cpu() == v[20].to(torch.float8_e4m3fn).bfloat16()).all()
    want = q[:, 0, 3].double().cpu() * 448 * 2.0 ** exponent / 8
    assert ((lse[:, 0].double().cpu() - want).abs() <= want * 2.0 ** -21).all()      # at most eight roundings of 32 bits


@pytest.mark.parametrize("rows", [1, 16])
def test_large_queries_over_keys_of_the_smallest_scales(sv, rows):  # noqa: F811
    """2^127 times 448 leaves 32 bits before a key's scale of 2^-100 is applied, the score does not"""
    large_scores(sv, rows, -100)


@pytest.mark.parametrize("exponent", [-100, -60, -20])
@pytest.mark.parametrize("rows", [1, 16, 40, 150])
def test_scores_beyond_the_range_of_an_exponential(sv, rows, exponent):  # noqa: F811
    """of 2^26 to 2^113"""
    large_scores(sv, rows, exponent)


def test_infinite_queries_over_8_bit_keys(sv):  # noqa: F811
    """give what they give over others: no value, and the logarithm of a sum of zeros"""
    for form in FORMS:
        cache, batch, q, n, kv = infinite_query("e4m3", form, sv)
        out, lse = sv.paged_attention(cache, batch, q, with_lse=True)
        assert torch.isnan(out[0, 0]).all() and float(lse[0, 0]) == -math.inf and torch.isfinite(out[0, 1]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,history,biases", [(2, 1000, 30, 129), (1, 5000, 0, 5000), (3, 9000, 100, 3001), (700, 1000, 20, 600), (400, 3001, 9000, 700), (2, 50, 5, 4096), (150, 33001, 500, 2000)])
def test_long_lists_of_biases(sv, rows, vocab, history, biases, dtype):  # noqa: F811
    """as long as the vocabulary and longer, the same id many times: sums in the order of the list, whatever the call's size"""
    gen = torch.Generator().manual_seed(rows + vocab)
    x = (torch.randn(rows, vocab, generator=gen) * 4).to(dtype).to(DEV)
    a = {"bias_ids": torch.randint(-2, vocab + 2, (rows, biases), generator=gen).int(), "bias": torch.randn(rows, biases, generator=gen) * 5,
         "mask": torch.randint(-2 ** 31, 2 ** 31, (rows, (vocab + 31) // 32), generator=gen).int()}
    a["bias_ids"][:, biases // 2:] %= max(1, vocab // 3)
    if history:
        a["tokens"] = torch.randint(0, vocab, (rows, history), generator=gen).int()
        a["repetition"], a["frequency"] = 1 + torch.rand(rows, generator=gen), torch.rand(rows, generator=gen)
    dev = {k: v.to(DEV) for k, v in a.items()}
    got = sv.logits_process(x, **dev)
    some = sorted({0, rows // 2, rows - 1})
    want, tol = ref.logits(x[some], **{k: v[some] for k, v in a.items()})
    tol = tol + (ref.F32_HALF if dtype == torch.float32 else ref.BF16_HALF) * (want.abs() + tol)
    fine, have = torch.isfinite(want), got[some].double().cpu()
    assert torch.equal(have[~fine], want[~fine]) and ((have - want).abs()[fine] <= tol[fine]).all()
    for r in some:
        part = slice(r, r + 1)
        assert torch.equal(got[part], sv.logits_process(x[part], **{k: v[part] for k, v in dev.items()}))
    assert sv.logits_process(x, out=x, **dev) is x and torch.equal(x, got)
    # one more entry than a short list may have, the last without weight: the same sums
    short = {"bias_ids": dev["bias_ids"][:, :128].contiguous(), "bias": dev["bias"][:, :128].contiguous()}
    longer = {"bias_ids": torch.cat([short["bias_ids"], torch.full((rows, 1), -1, dtype=torch.int32, device=DEV)], 1), "bias": torch.cat([short["bias"], torch.ones(rows, 1, device=DEV)], 1)}
    assert torch.equal(sv.logits_process(got, **short), sv.logits_process(got, **longer))


def test_windows_and_sizes_beyond_32_bits(sv, ofa, monkeypatch):  # noqa: F811
    cache, batch, gen = make(sv, [4], [60], 1, 64, 16)
    q = queries(gen, 4, 2, 64)
    want = sv.paged_attention(cache, batch, q)
    for fast in (True, False):
        if not fast:
            monkeypatch.setattr(sv, "_fast_module", None)
        for window in (2 ** 31, 2 ** 32 + 5, 2 ** 40):
            assert torch.equal(sv.paged_attention(cache, batch, q, window=window), want)
        many = 2 ** 32 + 4
        k, x = torch.zeros(1, 1, 64, dtype=torch.bfloat16, device=DEV).expand(many, -1, -1), torch.zeros(1, 8, device=DEV).expand(many, -1)
        for bad in (lambda: sv.paged_attention(cache, batch, q, window=-2 ** 40), lambda: sv.kv_append(cache, batch, k, k), lambda: sv.kv_read(cache, batch, k=k, v=k),
                    lambda: sv.logits_process(x, out=x), lambda: sv.KVCache(k[None], k[None]), lambda: sv.KVBatch(i32([0] * 3), i32([1, 1]), i32([[0]]).expand(many, 1))):
            with pytest.raises(ofa.OfaError):
                bad()


def test_rows_that_a_sequence_is_too_short_for(sv):  # noqa: F811
    """are not kept, and that is said; sequences of length 0 are places that a padded batch does not use"""
    cache, batch, gen = make(sv, [6, 2], [4, 2], 1, 64, 8)
    k = torch.randn(8, 1, 64, generator=gen).bfloat16().to(DEV)
    before, idle = cache.k.clone(), sv.KVBatch(batch.q_start, i32([0, 0]), batch.pages, status=i32([0]))
    sv.kv_append(cache, idle, k, k)
    assert int(idle.status) == 0 and torch.equal(cache.k, before)
    sv.kv_append(cache, batch, k, k)
    assert int(batch.status) == sv.BAD_LENGTH
    batch.status.zero_()
    back, _ = sv.kv_read(cache, batch, 8)
    assert int(batch.status) == 0 and (back[:2] == 0).all() and torch.equal(back[2:], k[2:])


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
@pytest.mark.parametrize("rows", [1, 8, 40, 150])
def test_the_smallest_scales(sv, rows, dtype):  # noqa: F811
    """scores of order one from large queries and a scale below 1e-30"""
    cache, batch, gen = make(sv, [rows], [170], 1, 64, 16, dtype, max_new=rows)
    q = (torch.randn(rows, 2, 64, generator=gen) * 2.0 ** 112).bfloat16().to(DEV)
    for scale in (2.0 ** -115, -2.0 ** -115):
        check_attention(sv, cache, batch, q, scale=scale)
    out = sv.paged_attention(cache, batch, q, causal=False, scale=0.0)
    want = sv.kv_read(cache, sv.KVBatch(i32([0, 170]), i32([170]), batch.pages), 170)[1].double()[:, 0]
    assert ((out.double() - want.mean(0)).abs() <= (want.abs().mean(0) + want.mean(0).abs()) * ref.BF16_HALF * 1.01).all()


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
@pytest.mark.parametrize("order", ["rising", "falling", "any"])
@pytest.mark.parametrize("hints", [{}, {"max_kv": 6000}])
def test_scores_of_every_size_over_many_steps(sv, hints, order, dtype):  # noqa: F811
    """One dim alone counts, so that scores are exact: rows of 2^-4 to 2^100, of either sign, over keys that rise, fall and repeat; with a scale that is no power of two"""
    gen = torch.Generator().manual_seed(7)
    n, rows, dim = 6000, 150, 64
    k = torch.zeros(n, dim)
    x = torch.randn(n, generator=gen).to(torch.float8_e4m3fn).float() if dtype == "e4m3" else torch.randn(n, generator=gen).bfloat16().float()
    k[:, 3] = x if order == "any" else x.sort(descending=order == "falling").values
    v = torch.randn(n, dim, generator=gen)
    cache = held_cache(sv, [k, v], [torch.zeros(n)] * 2) if dtype == "e4m3" else sv.KVCache(k.bfloat16().view(1, 1, n, dim).to(DEV), v.bfloat16().view(1, 1, n, dim).to(DEV))
    q = torch.zeros(rows, 1, dim)
    q[:, 0, 3] = torch.exp2(torch.arange(rows) * 104 / (rows - 1) - 4) * (1 - 2 * (torch.arange(rows) % 2))
    q = q.bfloat16().to(DEV)
    batch = sv.KVBatch(i32([0, rows]), i32([n]), i32([[0]]), max_new=rows, **hints)
    for scale in (0.17, -0.17):
        out, lse = sv.paged_attention(cache, batch, q, causal=False, scale=scale, with_lse=True)
        s = q[:, 0, 3].double().cpu()[:, None] * k[:, 3].double() * C.c_float(scale).value
        want, p = torch.logsumexp(s, 1), torch.softmax(s, 1)
        held = cache.v[0, 0].double().cpu()
        # a score's exponent: the scale times log2 e and the product rounded (2^-23 of it), which moves a probability by as much of its distance from the largest
        off = (p * (s.max(1, keepdim=True).values - s)).sum(1)[:, None] * 2.0 ** -22 + 2.0 ** -18
        assert ((out[:, 0].double().cpu() - p @ held).abs() <= (p @ held.abs()) * (ref.BF16_HALF + 2 * off) + (p @ held).abs() * ref.BF16_HALF * 1.01 + 1e-37).all()
        assert ((lse[:, 0].double().cpu() - want).abs() <= want.abs() * 2.0 ** -21 + 2.0 ** -18).all()


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
@pytest.mark.parametrize("layout", ["two_pools", "by_page", "by_head", "by_row", "v_first"])
def test_keys_and_values_in_one_tensor(sv, layout, dtype):  # noqa: F811
    """and rows read into one: whatever lies beside one another is taken"""
    pages, heads, page, dim = 9, 2, 16, 64
    t = torch.bfloat16 if dtype == "bf16" else torch.float8_e4m3fn

    def pair(last, t):
        both = {"two_pools": (2, pages, heads, page, *last), "v_first": (2, pages, heads, page, *last), "by_page": (pages, 2, heads, page, *last), "by_head": (pages, heads, 2, page, *last),
                "by_row": (pages, heads, page, 2, *last)}[layout]
        x = torch.zeros(both, dtype=torch.uint8 if t != torch.bfloat16 else t, device=DEV)
        x = x.view(t) if t != torch.uint8 else x
        axis = {"two_pools": 0, "v_first": 0, "by_page": 1, "by_head": 2, "by_row": 3}[layout]
        k, v = x.select(axis, 0), x.select(axis, 1)
        return (v, k) if layout == "v_first" else (k, v)
    k, v = pair((dim,), t)
    cache = sv.KVCache(k, v, *(pair((), torch.uint8) if dtype == "e4m3" else ()))
    plain = sv.KVCache.empty(pages, page, heads, dim, dtype)
    gen = torch.Generator().manual_seed(1)
    rows = torch.randn(100, 2, 2, dim, generator=gen).bfloat16().to(DEV)
    batch = sv.KVBatch(i32([0, 100]), i32([100]), i32([[4, 2, 8, 0, 1, 3, 7]]))
    for c in (cache, plain):
        sv.kv_append(c, batch, rows[:, 0], rows[:, 1])
    into = torch.zeros(100, 2, 3, dim, dtype=torch.bfloat16, device=DEV)
    got, want = sv.kv_read(cache, batch, k=into[:, :, 0], v=into[:, :, 2]), sv.kv_read(plain, batch, 100)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and not into[:, :, 1].any()
    q = queries(gen, 100, 4, dim)
    assert torch.equal(sv.paged_attention(cache, batch, q), sv.paged_attention(plain, batch, q))
