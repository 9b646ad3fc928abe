"""Calls of the cache operators at the edges of what they allow, on the GPU, against the formula in 64 bits."""
import math

import pytest
import torch

import cache_reference as R
import sageattention as S
from sageattention import cache as C
from test_gpu_cache_attention import _check            # a call against the formula, with that file's bound

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _seed():
    torch.manual_seed(0)


# ---- rotary ------------------------------------------------------------------------------------------------------

def _turned(x, pos, rotary, backward=False):
    return R.rotate(x.transpose(0, 1), pos, rotary.inv_freq, rotary.magnitude, rotary.interleaved, backward).transpose(0, 1)


def _rot_close(got, want, x):
    """Angles to 2^-24 of pi, products and sums in fp32: 2^-21 of the pair's length at most; half a step of the output."""
    eps = torch.finfo(got.dtype).eps / 2
    size = x.double().abs().amax(-1, keepdim=True) * 1.5 * 1.42
    assert ((got.double() - want).abs() <= eps * want.abs() + 2.0 ** -21 * size + torch.finfo(got.dtype).tiny * eps).all()


@pytest.mark.parametrize("fresh_first", [True, False])
def test_a_part_of_a_fused_projection_turned_fresh_and_in_place(fresh_first):
    """One SageRotary, one strided q alone: fresh outputs are packed, those in place have the projection's strides."""
    rotary, pos = S.SageRotary(64), torch.arange(100, 137, device="cuda")
    qkv = torch.randn((37, 8, 64), device="cuda").half()
    for fresh in (fresh_first, not fresh_first, fresh_first):
        before = qkv.clone()
        q = qkv[:, 2:6]
        # on the host first: a plan of the other form would write with the other form's strides
        key_out = None if fresh else q
        words = C._plan_rotary(q, None, pos, rotary, "HND", key_out)
        kept = [p for k, p in rotary._plans.items() if (k[-1] is None) == fresh]
        assert all(p == words for p in kept) and C._plan_rotary(q, None, pos, rotary, "HND", None) != C._plan_rotary(q, None, pos, rotary, "HND", q)
        got = S.sage_rotary(q, None, pos, rotary, out=key_out)
        _rot_close(got, _turned(before[:, 2:6], pos, rotary), before[:, 2:6])
        assert torch.equal(qkv[:, :2], before[:, :2]) and torch.equal(qkv[:, 6:], before[:, 6:])
        assert got.is_contiguous() if fresh else got is q
        if fresh:
            assert torch.equal(qkv, before)


def test_one_tensor_as_both_inputs_is_not_turned_in_place_twice():
    rotary, pos = S.SageRotary(64), torch.arange(9, device="cuda")
    q = torch.randn((9, 2, 64), device="cuda").half()
    a, b = S.sage_rotary(q, q, pos, rotary)
    assert torch.equal(a, b)
    with pytest.raises(ValueError, match="overlaps"):
        S.sage_rotary(q, q, pos, rotary, out=(q, q))


@pytest.mark.parametrize("layout", ["HND", "NHD"])
def test_packed_and_batched_tensors_do_not_mix(layout):
    rotary, pos = S.SageRotary(64), torch.arange(5, device="cuda")
    packed = torch.randn((5, 2, 64), device="cuda").half()
    batched = packed[None] if layout == "NHD" else packed.transpose(0, 1)[None]
    for q, k in ((packed, batched), (batched, packed)):
        with pytest.raises(ValueError, match="both"):
            S.sage_rotary(q, k, pos, rotary, tensor_layout=layout)
    want = S.sage_rotary(packed, None, pos, rotary)
    got = S.sage_rotary(batched, batched, pos, rotary, tensor_layout=layout)
    for x in got:
        assert torch.equal(x[0] if layout == "NHD" else x[0].transpose(0, 1), want)


def test_gradients_at_any_offset():
    """The gradient of a part of something larger, behind an odd number of elements: against the formula."""
    rotary, pos = S.SageRotary(64, rotary_dim=32), torch.arange(7, 18, device="cuda")
    q = torch.randn((11, 3, 64), device="cuda").half().requires_grad_()
    odd = torch.randn(3, device="cuda").half().requires_grad_()
    y = torch.cat([odd, S.sage_rotary(q, None, pos, rotary).flatten()])
    g = torch.randn_like(y)
    y.backward(g)
    g = g[3:].view(11, 3, 64)
    _rot_close(q.grad, _turned(g, pos, rotary, backward=True), g)


def test_a_training_step_is_captured_and_replayed():
    """Forward and backward in one graph, warmed up on its stream; replays follow what the inputs and positions hold by then."""
    rotary = S.SageRotary(64, rotary_dim=48, scaling="parts", factor=4.0)
    q, k = (torch.randn((13, h, 64), device="cuda").bfloat16().requires_grad_() for h in (4, 2))
    pos, g = torch.arange(13, device="cuda"), [torch.randn((13, h, 64), device="cuda").bfloat16() for h in (4, 2)]
    step = lambda: torch.autograd.grad(S.sage_rotary(q, k, pos, rotary), (q, k), g)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        grads = step()
    for _ in range(2):
        pos.add_(1000)
        for x in g:
            x.copy_(torch.randn_like(x))
        graph.replay()
        torch.cuda.synchronize()
        for got, x in zip(grads, g):
            _rot_close(got, _turned(x, pos, rotary, backward=True), x)


# ---- writing -----------------------------------------------------------------------------------------------------

def test_autograd_learns_of_writes_to_the_cache():
    cache = S.SageCache.empty(2, 16, 2, 64)
    x, slots = torch.randn((3, 2, 64), device="cuda").half(), torch.arange(3, device="cuda")
    w = torch.ones_like(cache.v_scale, requires_grad=True)
    y = (w * cache.v_scale).sum()
    S.sage_cache_write(cache, x, x, slots)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        served = S.SageCache.empty(2, 16, 2, 64)
    S.sage_cache_write(served, x, x, slots)          # tensors of inference mode have no versions
    assert torch.equal(served.k_scale, cache.k_scale) and torch.equal(served.v_scale, cache.v_scale)


@pytest.mark.parametrize("d", [40, 72, 128])
def test_the_shift_of_a_cache_is_a_copy_in_the_shape_it_was_given(d):
    import copy
    shift = torch.randn((2, d), device="cuda", requires_grad=True)
    cache = S.SageCache.empty(2, 16, 2, d, k_shift=shift)
    assert cache.k_shift.shape == (2, d) and torch.equal(cache.k_shift, shift) and not cache.k_shift.requires_grad
    k, slots = torch.randn((20, 2, d), device="cuda").half(), torch.arange(20, device="cuda")
    twin = S.SageCache(*(torch.zeros_like(t) for t in (cache.k_codes, cache.k_scale, cache.v_codes, cache.v_scale)), d, cache.k_shift)
    want = shift.detach().clone()
    with torch.no_grad():
        shift.zero_()
    for c in (cache, twin, copy.deepcopy(cache)):
        assert torch.equal(c.k_shift, want)
        S.sage_cache_write(c, k, k, slots)
        codes, scale = R.quantise(k.float() - want, True)
        assert torch.equal(c.k_codes.transpose(1, 2).flatten(0, 1)[:20, :, :d].double(), codes) and (c.k_codes[..., d:] == 0).all()
        assert torch.equal(c.k_scale.transpose(1, 2).flatten(0, 1)[:20], scale)


# ---- attention ---------------------------------------------------------------------------------------------------

def _setup(lens, t, hq=8, hkv=2, d=128, page=16, dtype=torch.float16, int8=True, shift=False, seed=0):
    """Sequences of those lengths in scattered pages, written; queries of t new tokens each."""
    gen = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    k_shift = 0.5 * torch.randn((hkv, d), generator=gen).cuda() if shift else None
    cache = S.SageCache.empty(sum(need) + 3, page, hkv, d, dtype=dtype, int8=int8, k_shift=k_shift)
    table = torch.full((len(lens), max(need) + 1), -1, dtype=torch.int32)
    order, at = torch.randperm(cache.num_pages, generator=gen).int(), 0
    for i, m in enumerate(need):
        table[i, :m] = order[at:at + m]
        at += m
    k, v = (torch.randn((sum(lens), hkv, d), generator=gen).to(dtype).cuda() for _ in range(2))
    S.sage_cache_write(cache, k, v, torch.cat([_slots(cache, table, i, torch.arange(n)) for i, n in enumerate(lens)]).cuda())
    q = torch.randn((len(lens) * t, hq, d), generator=gen).to(dtype).cuda()
    return cache, table.cuda(), q, torch.tensor(lens, dtype=torch.int32).cuda(), gen


def _slots(cache, table, i, at):
    return table[i, at // cache.page_size].long() * cache.page_size + at % cache.page_size


# New tokens x 4 query heads: one and two row tiles of the kernel for few rows, both forms of the kernel for many.
ROWS = [1, 3, 6, 12, 40]


@pytest.mark.parametrize("lens", [(230, 150), (9000, 40)])            # the longer ones are cut and joined
@pytest.mark.parametrize("which", ["k", "v", "both"])
@pytest.mark.parametrize("t", ROWS)
def test_a_nan_in_one_of_key_and_value(t, which, lens):
    """A row that sees it is NaN; its LSE is NaN for K, and for V alone that of the scores; no other row changes a bit."""
    cache, table, q, lens_d, gen = _setup(lens, t, dtype=torch.bfloat16)
    mask = torch.eye(t, dtype=torch.bool).repeat(2, 1).cuda()
    call = lambda: S.sageattn_cached(q, cache, table, lens_d, tree_mask=mask, return_lse=True)
    k, v = (torch.randn((1, 2, 128), generator=gen).cuda().bfloat16() for _ in range(2))
    slot = _slots(cache, table.cpu(), 0, torch.tensor([lens[0] - 1])).cuda()          # the last draft of the first sequence, which that alone sees
    S.sage_cache_write(cache, k, v, slot)
    clean, clean_lse = call()
    if which != "v":
        k[0, 0, 3] = math.nan
    if which != "k":
        v[0, 0, 100] = -math.inf
    S.sage_cache_write(cache, k, v, slot)
    out, lse = call()
    hit = torch.zeros((2 * t, 8), dtype=torch.bool, device="cuda")
    hit[t - 1, :4] = True                            # (query heads 0-3 share K/V head 0)
    assert torch.isnan(out[hit]).all()
    assert torch.equal(out[~hit], clean[~hit]) and torch.equal(lse[~hit], clean_lse[~hit])
    if which == "v":                                 # the same scores; the fp32 sum over the scale of V takes other roundings
        assert ((lse - clean_lse)[hit].abs() <= 2e-5 * clean_lse[hit].abs().clamp(min=1)).all()
    else:
        assert torch.isnan(lse[hit]).all()


# One key whose weight dwarfs that of each of the others, which together still count: 262 144 of them at 2^-25.2.  Units are
# not cut (there are more than the GPU has places for, all of them over the same two pages), so that a row's maximum
# is that key's throughout.
def _dominated(t, n_seq, n=262144, d=128, hkv=8, page=256):
    cache = S.SageCache.empty(2, page, hkv, d, int8=True)
    k, v = torch.zeros((2 * page, hkv, d), dtype=torch.float16, device="cuda"), torch.ones((2 * page, hkv, d), dtype=torch.float16, device="cuda")
    k[0] = 1.544                                     # times 1 / sqrt(128) and log2(e), over 128 columns: 25.2
    S.sage_cache_write(cache, k, v, torch.arange(2 * page, device="cuda"))
    table = torch.ones((1, n // page), dtype=torch.int32, device="cuda")
    table[0, 0] = 0
    q = torch.ones((n_seq * t, 4 * hkv, d), dtype=torch.float16, device="cuda")
    lens = torch.full((n_seq,), n, dtype=torch.int32, device="cuda")
    top = (cache.k_codes[0, 0, 0].double() * cache.k_scale[0, 0, 0].double()).sum() * d ** -0.5
    row = torch.arange(t, device="cuda").repeat(n_seq)
    others = (n - t + row).double()                  # keys of weight 1 that the row sees beside the first
    lse = torch.logaddexp(top, others.log())
    return cache, table.expand(n_seq, -1), q, lens, lse[:, None].expand(-1, 4 * hkv)


DOMINATED = [(1, 160), (6, 160), (12, 40), (40, 40)]


@pytest.mark.parametrize("t,n_seq", DOMINATED)
def test_small_weights_beside_a_dominant_one(t, n_seq):
    """Values of 1: every output is 1.  A weight is off by 2^-11 of itself, or by 2^-25 where fp16 is subnormal, and the row's
    largest stands at 2^4 at least: 2^-29 of it per key.  The matrix instructions add 16 keys at a time to an fp32 accumulator: 2^-23
    of the sum each time.  As above, 1.25 covers the fp32 parts beside these, and half a step is the output's."""
    n = 262144
    cache, table, q, lens, _ = _dominated(t, n_seq, n)
    out = S.sageattn_cached(q, cache, table, lens)
    off = (out.double() - 1).abs().max().item()
    assert off <= 1.25 * 2.0 ** -11 + n * 2.0 ** -29 + n / 16 * 2.0 ** -23 + 2.0 ** -11, off


@pytest.mark.parametrize("t,n_seq", DOMINATED)
def test_the_sum_of_small_weights_beside_a_dominant_one(t, n_seq):
    """The LSE's bound is that of every other call: 2e-5 max(1, |lse|)."""
    cache, table, q, lens, want = _dominated(t, n_seq)
    _, lse = S.sageattn_cached(q, cache, table, lens, return_lse=True)
    off = ((lse.double() - want).abs() / want.abs().clamp(min=1)).max().item()
    assert off <= 2e-5, off


@pytest.mark.parametrize("t", ROWS)
def test_rows_that_nothing_wrote(t):
    """Keys and values of zero: outputs of zero, an LSE of the keys' number, whatever is seen beside them."""
    cache = S.SageCache.empty(4, 64, 2, 128)
    q = torch.randn((t, 8, 128), device="cuda").half()
    table = torch.arange(4, dtype=torch.int32, device="cuda").repeat(1, 256)           # 65 536 keys
    for n in (t, 200, 65536):
        out, lse = S.sageattn_cached(q, cache, table, torch.tensor([n], dtype=torch.int32, device="cuda"), return_lse=True)
        want = (n - t + 1 + torch.arange(t, device="cuda")).double().log()[:, None]
        assert (out == 0).all() and ((lse.double() - want).abs() <= 2e-5 * want.clamp(min=1)).all()
    v = torch.full((1, 2, 128), 50000.0, dtype=torch.float16, device="cuda")
    S.sage_cache_write(cache, torch.zeros_like(v), v, torch.zeros(1, dtype=torch.int64, device="cuda"))
    out, lse = S.sageattn_cached(q, cache, table[:, :4], torch.tensor([256], dtype=torch.int32, device="cuda"), return_lse=True)
    n = (256 - t + 1 + torch.arange(t, device="cuda")).double()[:, None]
    assert ((lse.double() - n.log()).abs() <= 2e-5 * n.log()).all()
    value = 448.0 * cache.v_scale[0, 0, 0].item()
    assert ((out.double() - value / n[..., None]).abs() <= 1.25 * 2.0 ** -11 * value / n[..., None] + 2.0 ** -11 * value / n[..., None]).all()


# ---- every form of attention by kind of codes, page and width ------------------------------------------------------------
# e4m3 keys (the rule for bfloat16) and int8 ones, more than 32 and more than 128 rows per K/V head.

@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("d", [8, 40, 64, 72, 96, 128])
def test_many_rows_of_any_width_and_page(d, page):
    _check([300, 12, 77], [12, 5, 12], 4, 1, d, page, torch.bfloat16, False, tree=True, shift=True)
    _check([300, 41], [12, 12], 4, 1, d, page, torch.float16, True, shift=True)
    _check([290, 40], [40, 33], 4, 1, d, page, torch.float16, False, shift=True)
    _check([600], [40], 4, 1, d, page, torch.bfloat16, True, tree=True, shift=True)


@pytest.mark.parametrize("int8", [True, False])
@pytest.mark.parametrize("t", ROWS)
def test_long_sequences_that_are_cut_and_joined(t, int8):
    _check([7000, 90, 3001], [t, t, max(1, t // 3)], 8, 2, 128, 32, torch.bfloat16, int8, tree=True)
    _check([5003], [t], 4, 1, 64, 128, torch.float16, int8, shift=True)


@pytest.mark.parametrize("batch,t", [(160, 3), (120, 6), (90, 12), (40, 40)])
def test_many_short_sequences_of_e4m3_keys(batch, t):
    """More units than places: most of them whole, some cut."""
    lens = [(37 * i) % 90 + (t if i % 5 else 0) for i in range(batch)]
    _check(lens, [t if i % 4 else max(1, t // 2) for i in range(batch)], 16, 4, 64, 16, torch.bfloat16, False, tree=t % 2 == 1, shift=True)


@pytest.mark.parametrize("shift", [False, True])
@pytest.mark.parametrize("t", ROWS)
def test_padding_with_queries_of_anything(t, shift):
    """A sequence without keys, one whose pages do not exist and a token that its mask leaves nothing, with queries that
    are not finite: zeros and an LSE of -infinity."""
    for bad in (math.nan, math.inf):
        for n in (90, 3000):                         # whole units, and units that are cut
            cache, table, q, lens, _ = _setup((n, n + 1, n + 2), t, dtype=torch.bfloat16, shift=shift)
            mask = torch.ones((3 * t, t), dtype=torch.bool, device="cuda")
            want, want_lse = S.sageattn_cached(q, cache, table, lens, tree_mask=mask, return_lse=True)
            lens[1] = 0
            table[2] = -1
            q[t:] = bad
            out, lse = S.sageattn_cached(q, cache, table, lens, tree_mask=mask, return_lse=True)
            assert (out[t:] == 0).all() and (lse[t:] == -math.inf).all()
            assert torch.isfinite(lse[:t]).all() and ((lse - want_lse)[:t].abs() <= 4e-5 * want_lse[:t].abs().clamp(min=1)).all()
            lens[1] = t                              # only its own new tokens are cached, and masked
            mask[t:2 * t] = False
            out, lse = S.sageattn_cached(q, cache, table, lens, tree_mask=mask, return_lse=True)
            assert (out[t:] == 0).all() and (lse[t:] == -math.inf).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("t", ROWS)
def test_queries_that_are_not_finite(t, dtype):
    """NaN for the row, whatever the signs of its scores, and no bit of another row."""
    for n in (t, 200, 3000):
        cache, table, q, lens, _ = _setup((n, n + 5), t, dtype=dtype)
        mask = torch.eye(t, dtype=torch.bool, device="cuda").repeat(2, 1)
        want, want_lse = S.sageattn_cached(q, cache, table, lens, tree_mask=mask, return_lse=True)
        for at, value in (((0, 1, 5), math.inf), ((0, 2, 64), -math.inf), ((2 * t - 1, 6, 127), -math.inf), ((2 * t - 1, 7, 0), math.nan)):
            q[at] = value
        hit = ~torch.isfinite(q).all(-1)
        assert hit.sum() == 4
        out, lse = S.sageattn_cached(q, cache, table, lens, tree_mask=mask, return_lse=True)
        assert torch.isnan(out[hit]).all() and torch.isnan(lse[hit]).all()
        assert torch.equal(out[~hit], want[~hit]) and torch.equal(lse[~hit], want_lse[~hit])


@pytest.mark.parametrize("dtype,int8", [(torch.float16, True), (torch.bfloat16, False)])
def test_a_chunk_of_a_prompt_continues_a_cached_one(dtype, int8):
    """Many row tiles per sequence, as a chain: the way to go on with a prompt whose first part is cached."""
    _check([1600, 300, 257], [600, 1, 257], 2, 1, 128, 64, dtype, int8, shift=True)
    _check([700, 690], [700, 333], 3, 3, 72, 16, dtype, int8)


@pytest.mark.parametrize("t", ROWS)
def test_graphs_and_eager_calls_at_once(t):
    """Two graphs and eager calls on a third stream, all cut into parts, beside `sageattn` on a fourth: each its own bits."""
    calls = []
    for seed, lens in enumerate(((5000, 30), (3100, 2900), (9000, 17))):
        lens = tuple(max(n, t) for n in lens)
        cache, table, q, lens_d, _ = _setup(lens, t, seed=seed, shift=seed == 1)
        calls.append(lambda q=q, cache=cache, table=table, lens_d=lens_d: S.sageattn_cached(q, cache, table, lens_d, return_lse=True))
    x = [torch.randn((1, 8, 2048, 128), device="cuda").half() for _ in range(3)]
    calls.append(lambda: (S.sageattn(*x),))
    want = [[y.clone() for y in call()] for call in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for call, st in zip(calls[:2], streams):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            outs.append(call())
        graphs.append(graph)
    got = [[], []]
    for _ in range(10):
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        for i in (2, 3):
            with torch.cuda.stream(streams[i]):
                got[i - 2].append(calls[i]())
    torch.cuda.synchronize()
    for res, first in [(outs[0], want[0]), (outs[1], want[1])] + [(g, want[2]) for g in got[0]] + [(g, want[3]) for g in got[1]]:
        assert all(torch.equal(a, b) for a, b in zip(res, first))
