"""Attention over the quantised cache on the GPU, against the formula in 64 bits.

Tolerances.  Codes and scales are given, products of fp16 codes and fp16 queries are exact in the fp32 accumulator up to
its sums, so what is rounded to fewer bits is the weight of each value (fp16, 2^-11 relative, or 2^-25 of the row's
largest weight where that is more) and the output (2^-11 or 2^-8).  A weight off by 2^-11 moves an output row by at
most 2^-11 sum_j p_j |v_j|, which is at most 2^-11 max|v| in any column; the fp32 parts (scores of up to about 100
in the exponent: 100 x 2^-23, the approximate exponential 2^-22, the sums) stay below 2^-15 of the same; half of a
step is the rounding of the output itself.  So: |out - exact| <= 1.25 x 2^-11 max|v| + eps / 2 |exact|, with
max|v| over the keys of the head.  The LSE has only the fp32 parts: 2e-5 max(1, |lse|)."""
import math

import pytest
import torch

import cache_reference as R
import sageattention as S

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _seed():
    torch.manual_seed(0)


DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _make(lens, new, hq, hkv, d, page, dtype, int8, seed=0, shift=False, extra=3, width_extra=1):
    gen = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    pages = sum(need) + extra
    k_shift = 0.5 * torch.randn((hkv, d), generator=gen) if shift else None
    cache = S.SageCache.empty(pages, page, hkv, d, dtype=dtype, int8=int8, k_shift=None if k_shift is None else k_shift.cuda())
    order = torch.randperm(pages, generator=gen)
    table = torch.full((len(lens), max(need + [1]) + width_extra), -1, dtype=torch.int32)
    at = 0
    for i, m in enumerate(need):
        table[i, :m] = order[at:at + m].int()
        at += m
    total = sum(lens)
    k = (torch.randn((total, hkv, d), generator=gen) + (k_shift if shift else 0)).to(dtype).cuda()
    v = torch.randn((total, hkv, d), generator=gen).to(dtype).cuda()
    slots = torch.cat([table[i, torch.arange(n) // page].long() * page + torch.arange(n) % page for i, n in enumerate(lens)] + [torch.zeros(0, dtype=torch.long)])
    S.sage_cache_write(cache, k, v, slots.cuda())
    cu = [sum(new[:i]) for i in range(len(new) + 1)]
    q = torch.randn((cu[-1], hq, d), generator=gen).to(dtype).cuda()
    return cache, table.cuda(), q, cu, k_shift, gen


def _tree(new, gen, width=None):
    t = max(new)
    m = torch.zeros((sum(new), t if width is None else width), dtype=torch.bool)
    at = 0
    for n in new:
        for i in range(n):
            if i:
                m[at + i] = m[at + int(torch.randint(0, i, (1,), generator=gen))]
            m[at + i, i] = True
        at += n
    return m.cuda()


def _close(out, lse, want, want_lse, cache, lens, table):
    top = 0.0
    for i, n in enumerate(lens):
        if n:
            top = max(top, R.values(cache.v_codes, cache.v_scale, table[i], n, cache.head_dim)[0].abs().max().item())
    eps = torch.finfo(out.dtype).eps / 2
    off = (out.double() - want).abs()
    bound = 1.25 * 2.0 ** -11 * top + eps * want.abs()
    assert torch.isfinite(out).all()
    assert (off <= bound).all(), (off - bound).max().item()
    if lse is not None:
        assert torch.equal(torch.isinf(lse), torch.isinf(want_lse))
        fine = torch.isfinite(want_lse)
        assert ((lse.double() - want_lse)[fine].abs() <= 2e-5 * want_lse[fine].abs().clamp(min=1)).all()


def _check(lens, new, hq, hkv, d, page, dtype, int8, tree=False, shift=False, seed=0):
    cache, table, q, cu, k_shift, gen = _make(lens, new, hq, hkv, d, page, dtype, int8, seed, shift)
    mask = _tree(new, gen) if tree else None
    lens_d, cu_d = torch.tensor(lens, dtype=torch.int32).cuda(), torch.tensor(cu, dtype=torch.int32).cuda()
    out, lse = S.sageattn_cached(q, cache, table, lens_d, cu_d, max(new), tree_mask=mask, return_lse=True)
    torch.cuda.synchronize()
    want, want_lse = R.attend_cached(q, cache, table, lens, cu, mask, shift=None if k_shift is None else k_shift.cuda())
    _close(out, lse, want, want_lse, cache, lens, table)
    return out


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("int8", [True, False])
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 63, 64, 65, 129, 1000])
def test_one_token(n, int8, dtype):
    _check([n], [1], 4, 2, 128, 16, DT[dtype], int8)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("d", [8, 40, 64, 72, 96, 128])
def test_pages_and_widths(d, page):
    _check([300, 5, 257], [1, 1, 1], 6, 2, d, page, torch.float16, True, shift=True)
    _check([300, 5, 257], [3, 2, 4], 6, 2, d, page, torch.bfloat16, False, tree=True, shift=True)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (8, 8), (8, 1), (10, 2), (32, 8), (48, 48), (64, 4)])
def test_heads(hq, hkv):
    _check([200, 77], [1, 1], hq, hkv, 128, 32, torch.float16, True)
    _check([200, 77], [2, 5], hq, hkv, 128, 32, torch.bfloat16, True)


@pytest.mark.parametrize("t", [2, 3, 7, 8, 9, 16, 17, 31, 33, 64, 100])
@pytest.mark.parametrize("tree", [False, True])
def test_chains_and_trees(t, tree):
    _check([t, 200 + t, 1000], [t, max(1, t // 2), t], 8, 2, 128, 64, torch.float16, True, tree=tree)


def test_ragged_batch_with_empty_sequences():
    _check([500, 0, 3, 1300, 0, 64], [2, 1, 0, 4, 0, 3], 8, 4, 128, 16, torch.bfloat16, False)
    _check([500, 0, 3, 1300, 0, 64], [2, 1, 0, 4, 0, 3], 8, 4, 128, 16, torch.float16, True, tree=True)


def test_more_new_tokens_than_keys():
    _check([3, 40], [8, 6], 4, 2, 64, 16, torch.float16, True)
    _check([3, 40], [8, 6], 4, 2, 64, 16, torch.float16, True, tree=True)


@pytest.mark.parametrize("batch", [150, 400])
def test_many_sequences(batch):
    lens = [(37 * i) % 90 for i in range(batch)]
    _check(lens, [1 if i % 3 else 2 for i in range(batch)], 4, 2, 64, 16, torch.float16, True)


def test_long_sequence_is_split_and_joined():
    cache, table, q, cu, _, _ = _make([20000], [1], 8, 2, 128, 64, torch.float16, True)
    lens = torch.tensor([20000], dtype=torch.int32).cuda()
    out, lse = S.sageattn_cached(q, cache, table, lens, return_lse=True)
    want, want_lse = R.attend_cached(q, cache, table, [20000], cu)
    _close(out, lse, want, want_lse, cache, [20000], table)
    again = S.sageattn_cached(q, cache, table, lens)
    assert torch.equal(out, again)


def test_uniform_form_equals_packed_form():
    cache, table, q, cu, _, _ = _make([100, 300, 70], [2, 2, 2], 8, 2, 128, 16, torch.bfloat16, True)
    lens = torch.tensor([100, 300, 70], dtype=torch.int32).cuda()
    a = S.sageattn_cached(q, cache, table, lens)
    b = S.sageattn_cached(q, cache, table, lens, torch.tensor(cu, dtype=torch.int32).cuda(), 2)
    assert torch.equal(a, b)


def test_strided_views_and_out():
    cache, table, q, cu, _, _ = _make([100, 300], [3, 3], 8, 2, 128, 16, torch.float16, True)
    lens = torch.tensor([100, 300], dtype=torch.int32).cuda()
    want = S.sageattn_cached(q, cache, table, lens)
    wide = torch.zeros((6, 8, 3, 128), dtype=q.dtype, device="cuda")
    wide[:, :, 1] = q
    buf = torch.full((8, 9, 128), 7.0, dtype=q.dtype, device="cuda")
    res = S.sageattn_cached(wide[:, :, 1], cache, table, lens, out=buf[1:7, :8])
    assert res.data_ptr() == buf[1:7].data_ptr() and torch.equal(res, want)
    assert (buf[0] == 7).all() and (buf[7] == 7).all() and (buf[:, 8] == 7).all()


def test_rows_behind_the_last_sequence_stay():
    cache, table, q, cu, _, _ = _make([50, 60], [2, 1], 4, 2, 64, 16, torch.float16, True)
    lens = torch.tensor([50, 60], dtype=torch.int32).cuda()
    big = torch.cat([q, torch.full_like(q, math.nan)])
    out = torch.full_like(big, 5.0)
    S.sageattn_cached(big, cache, table, lens, torch.tensor(cu, dtype=torch.int32).cuda(), 2, out=out)
    assert torch.isfinite(out).all() and (out[3:] == 5).all() and not (out[:3] == 5).all()


def test_bad_pages_and_lengths_stay_in_bounds():
    """A page id outside the cache is a run of keys that nobody sees; lengths and starts are clamped."""
    cache, table, q, cu, _, _ = _make([200, 100], [1, 1], 4, 2, 128, 16, torch.float16, True)
    table[0, 3], table[0, 5], table[1, 0] = -5, 2 ** 31 - 1, cache.num_pages
    lens = torch.tensor([200, 100], dtype=torch.int32).cuda()
    out, lse = S.sageattn_cached(q, cache, table, lens, return_lse=True)
    want, want_lse = R.attend_cached(q, cache, table, [200, 100], cu)
    _close(out, lse, want, want_lse, cache, [200, 100], table)
    table[:] = -1
    out, lse = S.sageattn_cached(q, cache, table, torch.tensor([2 ** 30, -7], dtype=torch.int32).cuda(), return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    out = torch.full_like(q, 3.0)
    S.sageattn_cached(q, cache, table, lens, torch.tensor([-4, 2 ** 30, -9], dtype=torch.int32).cuda(), 1, out=out)
    assert torch.isfinite(out).all()


def test_what_a_mask_hides_reaches_nothing():
    """NaN and infinite keys and values of drafted tokens, seen by some rows and hidden from others."""
    cache, table, q, cu, _, gen = _make([130, 90], [6, 6], 8, 2, 128, 16, torch.bfloat16, True)
    mask = torch.eye(6, dtype=torch.bool).repeat(2, 1).cuda()
    lens = torch.tensor([130, 90], dtype=torch.int32).cuda()
    cu_d = torch.tensor(cu, dtype=torch.int32).cuda()
    clean = S.sageattn_cached(q, cache, table, lens, cu_d, 6, tree_mask=mask)
    bad = torch.randn((2, 2, 128), device="cuda").bfloat16()
    bad[0, 0, 3], bad[1, 1, 7] = math.nan, math.inf
    # draft 2 of the first sequence and draft 4 of the second
    slots = torch.tensor([table[0, 126 // 16] * 16 + 126 % 16, table[1, 88 // 16] * 16 + 88 % 16], device="cuda")
    S.sage_cache_write(cache, bad, bad, slots)
    out = S.sageattn_cached(q, cache, table, lens, cu_d, 6, tree_mask=mask)
    hit = torch.zeros((12, 8), dtype=torch.bool)
    hit[2, :4] = hit[6 + 4, 4:] = True               # (query heads 0-3 share K/V head 0)
    assert torch.isnan(out[hit.cuda()]).all()
    free = ~hit
    free[2] = free[10] = False                       # (those two tokens' own keys changed for all heads)
    assert torch.equal(out[free.cuda()], clean[free.cuda()])


def test_stale_rows_behind_the_length_reach_nothing():
    cache, table, q, cu, _, _ = _make([70], [1], 4, 2, 128, 64, torch.float16, False, width_extra=0)
    lens = torch.tensor([65], dtype=torch.int32).cuda()
    a = S.sageattn_cached(q, cache, table, lens)
    nan = torch.full((5, 2, 128), math.nan, dtype=torch.float16, device="cuda")
    S.sage_cache_write(cache, nan, nan, table[0, 1].long() * 64 + torch.arange(1, 6, device="cuda"))
    assert torch.equal(a, S.sageattn_cached(q, cache, table, lens))


def test_values_of_very_different_size():
    """The factor that keeps weights in fp16's range follows the largest seen: early outliers, late ones, and tiny values."""
    for factors in ([1e4, 1.0], [1.0, 1e4], [1e-6, 1e-6], [1.0, 1e-5]):
        cache, table, q, cu, _, gen = _make([512], [1], 4, 2, 128, 64, torch.bfloat16, True)
        v = torch.randn((512, 2, 128), generator=gen)
        v[:256] *= factors[0]
        v[256:] *= factors[1]
        k = torch.randn((512, 2, 128), generator=gen)
        slots = (table[0, torch.arange(512).cuda() // 64].long() * 64 + torch.arange(512).cuda() % 64)
        S.sage_cache_write(cache, k.bfloat16().cuda(), v.bfloat16().cuda(), slots)
        out, lse = S.sageattn_cached(q, cache, table, torch.tensor([512], dtype=torch.int32).cuda(), return_lse=True)
        want, want_lse = R.attend_cached(q, cache, table, [512], cu)
        # (each row against its own largest output column: every weight and code has 4 bits at least)
        off = (out.double() - want).abs().amax(-1) / want.abs().amax(-1)
        assert (off <= 2.0 ** -8 + 2.0 ** -9).all(), (factors, off.max().item())


@pytest.mark.parametrize("size", [1e-3, 1.0, 30.0])
def test_scores_of_any_size(size):
    """Flat and peaked softmaxes, and bf16 queries far outside fp16's range."""
    cache, table, q, cu, _, _ = _make([700], [2], 8, 2, 128, 32, torch.bfloat16, True)
    lens = torch.tensor([700], dtype=torch.int32).cuda()
    for up in (1.0, 2.0 ** 40, 2.0 ** -40):
        big = (q.float() * size * up).bfloat16()
        scale = 128 ** -0.5 / up
        out, lse = S.sageattn_cached(big, cache, table, lens, sm_scale=scale, return_lse=True)
        want, want_lse = R.attend_cached(big, cache, table, [700], cu, scale=scale)
        _close(out, lse, want, want_lse, cache, [700], table)


def test_captured_calls_have_their_own_workspace():
    cache, table, q, cu, _, _ = _make([3000, 900], [1, 1], 8, 2, 128, 64, torch.float16, True)
    lens = torch.tensor([3000, 900], dtype=torch.int32).cuda()
    q2 = torch.randn_like(q)
    want, want2 = S.sageattn_cached(q, cache, table, lens), S.sageattn_cached(q2, cache, table, lens)
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs, outs = [], []
    for x, st in zip((q, q2), side):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            S.sageattn_cached(x, cache, table, lens)
        st.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=st):
            outs.append(S.sageattn_cached(x, cache, table, lens))
        graphs.append(gr)
    for _ in range(20):
        for gr, st in zip(graphs, side):
            with torch.cuda.stream(st):
                gr.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want2)
    lens.fill_(100)                                  # lengths are read on the device by every replay
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], S.sageattn_cached(q, cache, table, lens))


def test_two_streams_at_once():
    cache, table, q, cu, _, _ = _make([5000], [1], 8, 2, 128, 64, torch.float16, True)
    lens = torch.tensor([5000], dtype=torch.int32).cuda()
    qs = [torch.randn_like(q) for _ in range(2)]
    want = [S.sageattn_cached(x, cache, table, lens) for x in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(S.sageattn_cached(qs[i], cache, table, lens))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_page_of_a_cache_beyond_32_bits():
    """Row offsets past 2^31 bytes: the last pages of a cache of 5 GB."""
    pages = 2 ** 31 // (8 * 256 * 128) + 40          # codes of K alone: 2.1e9 bytes
    cache = S.SageCache.empty(pages, 256, 8, 128)
    table = torch.arange(pages - 4, pages, dtype=torch.int32, device="cuda")[None]
    k, v = (torch.randn((1000, 8, 128), device="cuda").half() for _ in range(2))
    j = torch.arange(1000, device="cuda")
    S.sage_cache_write(cache, k, v, table[0, j // 256].long() * 256 + j % 256)
    q = torch.randn((1, 8, 128), device="cuda").half()
    out, lse = S.sageattn_cached(q, cache, table, torch.tensor([1000], dtype=torch.int32, device="cuda"), return_lse=True)
    want, want_lse = R.attend_cached(q, cache, table, [1000], [0, 1])
    _close(out, lse, want, want_lse, cache, [1000], table)
    cu = torch.tensor([0, 1000], dtype=torch.int32, device="cuda")
    k16, _ = S.sage_cache_read(cache, table, cu, 1000)
    # half a code's step of the row's largest / 127, then half a step of fp16 on the value that is read back
    top = k.float().abs().max()
    assert (k16.float() - k.float()).abs().max() <= top / 127 * 0.5 * (1 + 2.0 ** -20) + top * 2.0 ** -11


def test_sizes_given_as_tensors_are_read_each_time():
    cache, table, q, cu, _, _ = _make([40, 33], [4, 4], 8, 2, 64, 16, torch.float16, True)
    lens, cu = torch.tensor([40, 33], dtype=torch.int32, device="cuda"), torch.tensor(cu, dtype=torch.int32, device="cuda")
    count = torch.tensor(4)
    whole = S.sageattn_cached(q, cache, table, lens, cu, count, out=torch.full_like(q, 7.0))
    count.fill_(2)                                   # cut off behind the second new token of a sequence
    out = S.sageattn_cached(q, cache, table, lens, cu, count, out=torch.full_like(q, 7.0))
    assert torch.equal(out, S.sageattn_cached(q, cache, table, lens, cu, 2, out=torch.full_like(q, 7.0)))
    assert not torch.equal(out, whole)


def test_two_threads_on_one_stream():
    """Calls of both threads are cut into parts that a second kernel joins: neither may join the other's."""
    import threading
    cases = []
    for i in range(4):
        n = 9000 + 700 * i
        cache, table, q, _, _, _ = _make([n], [1 + 6 * (i % 2)], 8, 2, 128, 64, torch.float16, True, seed=i)
        cases.append((q, cache, table, torch.tensor([n], dtype=torch.int32, device="cuda")))
    call = lambda c: S.sageattn_cached(*c)
    want = [call(c) for c in cases]
    torch.cuda.synchronize()
    wrong = []

    def work(mine):
        for n in range(150):
            i = mine[n % len(mine)]
            out = call(cases[i])
            if not torch.equal(out, want[i]):
                wrong.append(i)
    threads = [threading.Thread(target=work, args=(m,)) for m in ((0, 1), (2, 3), (1, 2))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


# Rows (new tokens x 4 query heads) for one and for two row tiles of the kernel for few rows, and for either form of the
# kernel for many.
MANY = [3, 6, 12, 40]


@pytest.mark.parametrize("t", MANY)
def test_a_mask_hides_at_any_number_of_rows(t):
    cache, table, q, cu, _, gen = _make([230, 150], [t, t], 8, 2, 128, 16, torch.bfloat16, True, shift=True)
    mask = torch.eye(t, dtype=torch.bool).repeat(2, 1).cuda()
    lens, cu_d = torch.tensor([230, 150], dtype=torch.int32).cuda(), torch.tensor(cu, dtype=torch.int32).cuda()
    call = lambda: S.sageattn_cached(q, cache, table, lens, cu_d, t, tree_mask=mask, return_lse=True)
    clean, clean_lse = call()
    bad = torch.randn((2, 2, 128), generator=gen).cuda().bfloat16()
    bad[0, 0, 3], bad[1, 1, 7] = math.nan, math.inf
    # draft 1 of the first sequence, the last of the second
    at = (230 - t + 1, 149)
    slots = torch.tensor([int(table[i, n // 16]) * 16 + n % 16 for i, n in enumerate(at)], device="cuda")
    S.sage_cache_write(cache, bad, bad, slots)
    out, lse = call()
    hit = torch.zeros((2 * t, 8), dtype=torch.bool)
    hit[1, :4] = hit[2 * t - 1, 4:] = True           # (query heads 0-3 share K/V head 0)
    assert torch.isnan(out[hit.cuda()]).all()
    free = ~hit
    free[1] = free[2 * t - 1] = False                # (those two tokens' own keys changed for all heads)
    assert torch.equal(out[free.cuda()], clean[free.cuda()]) and torch.equal(lse[free.cuda()], clean_lse[free.cuda()])


@pytest.mark.parametrize("t", MANY)
def test_bad_pages_and_lengths_at_any_number_of_rows(t):
    cache, table, q, cu, _, _ = _make([300, 170], [t, t], 8, 2, 64, 16, torch.float16, True)
    table[0, 3], table[0, 9], table[1, 0] = -5, 2 ** 31 - 1, cache.num_pages
    lens, cu_d = torch.tensor([300, 170], dtype=torch.int32).cuda(), torch.tensor(cu, dtype=torch.int32).cuda()
    out, lse = S.sageattn_cached(q, cache, table, lens, return_lse=True)
    want, want_lse = R.attend_cached(q, cache, table, [300, 170], cu)
    _close(out, lse, want, want_lse, cache, [300, 170], table)
    out, lse = S.sageattn_cached(q, cache, torch.full_like(table, -1), torch.tensor([2 ** 30, -7], dtype=torch.int32).cuda(), cu_d, t, return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    out = S.sageattn_cached(q, cache, table, lens, torch.tensor([-4, 2 ** 30, -9], dtype=torch.int32).cuda(), t, out=torch.full_like(q, 3.0))
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("t", MANY)
def test_stale_and_unwritten_rows_at_any_number_of_rows(t):
    cache, table, q, _, _, _ = _make([200], [t], 8, 2, 128, 64, torch.float16, False, width_extra=0)
    lens = torch.tensor([130], dtype=torch.int32).cuda()
    a = S.sageattn_cached(q, cache, table, lens)
    nan = torch.full((62, 2, 128), math.nan, dtype=torch.float16, device="cuda")
    S.sage_cache_write(cache, nan, nan, table[0, 2].long() * 64 + torch.arange(2, 64, device="cuda"))
    assert torch.equal(a, S.sageattn_cached(q, cache, table, lens))
    empty = S.SageCache.empty(4, 64, 2, 128)         # nothing written: keys and values of zero
    out = S.sageattn_cached(q, empty, torch.arange(4, dtype=torch.int32, device="cuda").view(1, 4), lens)
    assert (out == 0).all()


@pytest.mark.parametrize("t", MANY)
def test_values_of_different_size_at_any_number_of_rows(t):
    for factors in ([1e4, 1.0], [1.0, 1e4], [1e-6, 1e-6], [1.0, 1e-5]):
        cache, table, q, cu, _, gen = _make([512], [t], 8, 2, 128, 64, torch.bfloat16, True)
        k, v = torch.randn((512, 2, 128), generator=gen), torch.randn((512, 2, 128), generator=gen)
        v[:200] *= factors[0]
        v[200:] *= factors[1]
        at = torch.arange(512, device="cuda")
        S.sage_cache_write(cache, k.bfloat16().cuda(), v.bfloat16().cuda(), table[0, at // 64].long() * 64 + at % 64)
        out = S.sageattn_cached(q, cache, table, torch.tensor([512], dtype=torch.int32).cuda())
        want, _ = R.attend_cached(q, cache, table, [512], cu)
        # (each row against its own largest output column: every weight and code has 4 bits at least)
        off = (out.double() - want).abs().amax(-1) / want.abs().amax(-1)
        assert (off <= 2.0 ** -8 + 2.0 ** -9).all(), (factors, off.max().item())


@pytest.mark.parametrize("t", MANY)
def test_views_and_rows_behind_at_any_number_of_rows(t):
    cache, table, q, cu, _, _ = _make([100, 300], [t, t], 8, 2, 72, 16, torch.float16, True)
    lens, cu_d = torch.tensor([100, 300], dtype=torch.int32).cuda(), torch.tensor(cu, dtype=torch.int32).cuda()
    want = S.sageattn_cached(q, cache, table, lens)
    wide = torch.full((2 * t + 3, 8, 3, 72), math.nan, dtype=q.dtype, device="cuda")
    wide[:2 * t, :, 1] = q
    buf = torch.full((2 * t + 3, 9, 72), 7.0, dtype=q.dtype, device="cuda")
    S.sageattn_cached(wide[:, :, 1], cache, table, lens, cu_d, t, out=buf[:, :8])
    assert torch.equal(buf[:2 * t, :8], want) and (buf[2 * t:] == 7).all() and (buf[:, 8] == 7).all()


@pytest.mark.parametrize("batch,t", [(400, 1), (300, 3), (120, 6), (90, 12), (40, 40)])
def test_many_sequences_of_many_rows(batch, t):
    lens = [(37 * i) % 90 + (t if i % 5 else 0) for i in range(batch)]
    _check(lens, [t if i % 4 else max(1, t // 2) for i in range(batch)], 16, 4, 64, 16, torch.float16, True, tree=t % 2 == 0)


def test_first_call_of_a_signature_is_captured_and_replayed():
    """Nothing of a call needs an earlier eager one; replays read what the tensors hold by then."""
    cache, table, q, cu, _, gen = _make([300, 77], [2, 2], 8, 2, 128, 16, torch.float16, True)
    lens = torch.tensor([300, 77], dtype=torch.int32).cuda()
    rotary = S.SageRotary(128)
    pos = torch.tensor([298, 299, 75, 76]).cuda()
    k, v = (torch.randn((4, 2, 128), generator=gen).half().cuda() for _ in range(2))
    slots = torch.tensor([int(table[i, n // 16]) * 16 + n % 16 for i, n in ((0, 298), (0, 299), (1, 75), (1, 76))]).cuda()
    cu_k = torch.tensor([0, 300, 377], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        qr, kr = S.sage_rotary(q, k, pos, rotary)
        S.sage_cache_write(cache, kr, v, slots)
        out, lse = S.sageattn_cached(qr, cache, table, lens, return_lse=True)
        back = S.sage_cache_read(cache, table, cu_k, 377)
    for _ in range(2):
        q.copy_(torch.randn(q.shape, generator=gen)); k.copy_(torch.randn(k.shape, generator=gen)); v.copy_(torch.randn(v.shape, generator=gen))
        graph.replay()
        torch.cuda.synchronize()
        qe, ke = S.sage_rotary(q, k, pos, rotary)
        S.sage_cache_write(cache, ke, v, slots)
        want, want_lse = S.sageattn_cached(qe, cache, table, lens, return_lse=True)
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
        whole = S.sage_cache_read(cache, table, cu_k, 377)
        assert torch.equal(back[0], whole[0]) and torch.equal(back[1], whole[1])


def test_a_copy_of_a_cache_is_its_own():
    import copy
    cache, table, q, _, _, gen = _make([90], [1], 8, 2, 72, 16, torch.float16, True, shift=True)
    lens = torch.tensor([90], dtype=torch.int32).cuda()
    rotary, pos = S.SageRotary(72), torch.tensor([89]).cuda()
    want, turned = S.sageattn_cached(q, cache, table, lens), S.sage_rotary(q, None, pos, rotary)
    twin, turn = copy.deepcopy(cache), copy.deepcopy(rotary)
    assert torch.equal(twin.k_shift, cache.k_shift) and torch.equal(S.sageattn_cached(q, twin, table, lens), want)
    x = torch.randn((90, 2, 72), generator=gen).half().cuda()
    at = torch.arange(90).cuda()
    S.sage_cache_write(twin, x, x, table[0, at // 16].long() * 16 + at % 16)
    assert not torch.equal(S.sageattn_cached(q, twin, table, lens), want)
    assert torch.equal(S.sageattn_cached(q, cache, table, lens), want)
    rotary.inv_freq.zero_()
    assert torch.equal(S.sage_rotary(q, None, pos, turn), turned) and torch.equal(S.sage_rotary(q, None, pos, rotary), q)
