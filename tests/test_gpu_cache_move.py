"""Writing to and reading from the quantised cache on the GPU, rotary positions, and the operators run together."""
import math

import pytest
import torch

import cache_reference as R
import sageattention as S
from sageattention import b200_backend as be

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _seed():
    torch.manual_seed(0)


DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _bits(t):
    return t.view(torch.uint8)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("int8", [True, False])
@pytest.mark.parametrize("d,page", [(128, 64), (128, 16), (96, 32), (64, 128), (40, 16), (8, 256)])
def test_write_gives_the_formula_s_codes(dtype, int8, d, page):
    gen = torch.Generator().manual_seed(d + page)
    tokens, heads = 333, 3
    shift = torch.randn((heads, d), generator=gen).cuda() if int8 else None
    cache = S.SageCache.empty(9 + 333 // page, page, heads, d, int8=int8, k_shift=shift)
    k, v = ((torch.randn((tokens, heads, d), generator=gen) * torch.rand((tokens, heads, 1), generator=gen).exp2() * 10).to(DT[dtype]).cuda() for _ in range(2))
    k[5], v[6] = 0, 0
    slots = torch.randperm(cache.num_pages * page, generator=gen)[:tokens].cuda()
    slots[7], slots[8] = -1, cache.num_pages * page          # left out
    S.sage_cache_write(cache, k, v, slots)
    live = torch.ones(tokens, dtype=torch.bool)
    live[7:9] = False
    x = k.float() if shift is None else k.float() - shift
    for codes, scale, rows, as_int8 in ((cache.k_codes, cache.k_scale, x, int8), (cache.v_codes, cache.v_scale, v.float(), False)):
        want_codes, want_scale = R.quantise(rows, as_int8)
        flat = codes.double().transpose(1, 2).flatten(0, 1)          # (slots, heads, width)
        flat_scale = scale.transpose(1, 2).flatten(0, 1)
        at = slots[live.cuda()]
        assert torch.equal(flat[at][..., :d], want_codes[live.cuda()])
        assert torch.equal(flat_scale[at], want_scale[live.cuda()])
        assert (flat[..., d:] == 0).all()
        rest = torch.ones(flat.shape[0], dtype=torch.bool, device="cuda")
        rest[at] = False
        assert (flat[rest] == 0).all() and (flat_scale[rest] == 0).all()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_write_gives_the_prologue_s_bits(dtype):
    """The same rows through the quantiser of `sageattn` and through the cache: the same codes and scales."""
    n, heads = 640, 2
    k, v = (torch.randn((1, heads, n, 128), device="cuda").to(DT[dtype]) for _ in range(2))
    pq = be.quant_qkv(k, k, v, smooth_k=False)
    cache = S.SageCache.empty(n // 64, 64, heads, 128, dtype=DT[dtype])
    S.sage_cache_write(cache, k[0].transpose(0, 1), v[0].transpose(0, 1), torch.arange(n, device="cuda"))
    order = be.k8_row_order(n, "cuda")
    assert torch.equal(_bits(cache.k_codes).transpose(0, 1).flatten(1, 2), _bits(pq["k8"])[:, order])
    assert torch.equal(cache.k_scale.transpose(0, 1).flatten(1), pq["sk"])
    assert torch.equal(_bits(cache.v_codes).transpose(0, 1).flatten(1, 2), _bits(pq["v8t"]).transpose(1, 2))
    assert torch.equal(cache.v_scale.transpose(0, 1).flatten(1), pq["sv"])


def test_write_int32_slots_strides_and_no_tokens():
    cache, other = S.SageCache.empty(4, 16, 2, 64), S.SageCache.empty(4, 16, 2, 64)
    kv = torch.randn((20, 3, 4, 64), device="cuda").half()
    k, v = kv[:, 0, ::2], kv[:, 2, 1::2]
    slots = torch.randperm(64)[:20].cuda()
    S.sage_cache_write(cache, k, v, slots)
    S.sage_cache_write(other, k.contiguous(), v.contiguous(), slots.int())
    S.sage_cache_write(other, k[:0], v[:0], slots[:0])
    assert torch.equal(_bits(cache.k_codes), _bits(other.k_codes)) and torch.equal(_bits(cache.v_codes), _bits(other.v_codes))
    assert torch.equal(cache.k_scale, other.k_scale) and torch.equal(cache.v_scale, other.v_scale)


@pytest.mark.parametrize("int8", [True, False])
@pytest.mark.parametrize("shift", [True, False])
def test_rows_that_are_not_finite(int8, shift):
    cache = S.SageCache.empty(2, 16, 2, 128, int8=int8, k_shift=torch.ones((2, 128), device="cuda") if shift else None)
    k, v = (torch.randn((8, 2, 128), device="cuda").bfloat16() for _ in range(2))
    k[1, 0, 5], k[2, 1, 127], k[3, 0, 0] = math.nan, math.inf, -math.inf
    v[4, 1, 64] = math.nan
    S.sage_cache_write(cache, k, v, torch.arange(8, device="cuda"))
    bad_k, bad_v = ~torch.isfinite(k).all(-1), ~torch.isfinite(v).all(-1)
    assert torch.equal(torch.isnan(cache.k_scale[0, :, :8]).T, bad_k) and torch.equal(torch.isnan(cache.v_scale[0, :, :8]).T, bad_v)
    assert torch.isfinite(cache.k_codes.float()).all() and torch.isfinite(cache.v_codes.float()).all()
    k16, v16 = S.sage_cache_read(cache, torch.zeros((1, 1), dtype=torch.int32, device="cuda"),
                                 torch.tensor([0, 8], dtype=torch.int32, device="cuda"), 8)
    assert torch.equal(torch.isnan(k16).all(-1), bad_k) and torch.equal(torch.isnan(k16).any(-1), bad_k)
    assert torch.equal(torch.isnan(v16).any(-1), bad_v)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("d,page,heads", [(128, 16, 3), (96, 64, 2), (64, 32, 5), (24, 256, 1)])
@pytest.mark.parametrize("lens", [[1], [100, 0, 17, 300], [0, 0, 64]])
def test_read_back(lens, d, page, heads, dtype):
    gen = torch.Generator().manual_seed(len(lens) + d)
    shift = torch.randn((heads, d), generator=gen).cuda() if d != 64 else None
    need = [-(-n // page) for n in lens]
    cache = S.SageCache.empty(sum(need) + 2, page, heads, d, int8=d != 96, k_shift=shift)
    table = torch.full((len(lens), max(need) + 1), -1, dtype=torch.int32)
    order, at = torch.randperm(cache.num_pages, generator=gen).int(), 0
    for i, m in enumerate(need):
        table[i, :m] = order[at:at + m]
        at += m
    total = sum(lens)
    slots = torch.cat([table[i, torch.arange(n) // page].long() * page + torch.arange(n) % page for i, n in enumerate(lens)])
    k, v = ((3 * torch.randn((total, heads, d), generator=gen)).to(DT[dtype]).cuda() for _ in range(2))
    S.sage_cache_write(cache, k, v, slots.cuda())
    cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32).cuda()
    buf = [torch.full((total + 5, heads + 1, d), 9.0, dtype=DT[dtype], device="cuda") for _ in range(2)]
    res = S.sage_cache_read(cache, table.cuda(), cu, total + 5, dtype=DT[dtype], out=tuple(x[:, :heads] for x in buf))
    fresh = S.sage_cache_read(cache, table.cuda(), cu, total, dtype=DT[dtype])
    at = 0
    for i, n in enumerate(lens):
        for j, (codes, scale) in enumerate(((cache.k_codes, cache.k_scale), (cache.v_codes, cache.v_scale))):
            ids = table[i, torch.arange(n) // page].long().cuda()
            off = (torch.arange(n) % page).cuda()
            c = codes.view(torch.uint8)[ids, :, off].view(codes.dtype).float()[..., :d]
            want = c * scale[ids, :, off][..., None]
            if j == 0 and shift is not None:
                want = want + shift
            assert torch.equal(res[j][at:at + n], want.to(DT[dtype])) and torch.equal(fresh[j][at:at + n], want.to(DT[dtype]))
        at += n
    for x in buf:
        assert (x[total:] == 9).all() and (x[:, heads] == 9).all()


def test_read_of_pages_that_do_not_exist():
    cache = S.SageCache.empty(3, 16, 2, 64, k_shift=torch.ones((2, 64), device="cuda"))
    x = torch.ones((48, 2, 64), device="cuda").half()
    S.sage_cache_write(cache, x, x, torch.arange(48, device="cuda"))
    table = torch.tensor([[0, -1, 2, 3]], dtype=torch.int32, device="cuda")
    k, v = S.sage_cache_read(cache, table, torch.tensor([0, 80], dtype=torch.int32, device="cuda"), 80)
    for t in (k, v):
        assert (t[:16] == 1).all() and (t[16:32] == 0).all() and (t[32:48] == 1).all() and (t[48:] == 0).all()
    out = (torch.full_like(k, 4.0), torch.full_like(v, 4.0))
    S.sage_cache_read(cache, table, torch.tensor([-100, 2 ** 31 - 1], dtype=torch.int32, device="cuda"), 80, out=out)
    S.sage_cache_read(cache, table, torch.tensor([70, 10], dtype=torch.int32, device="cuda"), 80, out=out)
    assert torch.isfinite(out[0]).all()


# ---- rotary ------------------------------------------------------------------------------------------------------
# The angle is exact to 2^-24 of a turn's pi, cosine, sine and the two products and their sum are fp32: 2^-21 of the
# pair's length at most; the rest is the rounding of the output.

def _rot_close(got, want, x):
    eps = torch.finfo(got.dtype).eps / 2
    size = x.double().abs().amax(-1, keepdim=True) * 1.5 * 1.42
    assert ((got.double() - want).abs() <= eps * want.abs() + 2.0 ** -21 * size + torch.finfo(got.dtype).tiny * eps).all()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rot", [(128, 128), (128, 64), (128, 32), (96, 96), (96, 72), (64, 8), (72, 72), (8, 8)])
def test_rotary(d, rot, interleaved, dtype):
    gen = torch.Generator().manual_seed(d + rot)
    for hq, hk, n in ((1, 1, 1), (5, 2, 37), (48, 48, 3)):
        q, k = (torch.randn((n, h, d), generator=gen).to(DT[dtype]).cuda() for h in (hq, hk))
        pos = torch.randint(0, 2 ** 31 - 1, (n,), generator=gen).cuda()
        pos[0] = 0
        rotary = S.SageRotary(d, rotary_dim=rot, interleaved=interleaved, scaling="parts", factor=4.0)
        for p in (pos, pos.int(), -pos):
            for back in (False, True):
                a, b = S.sage_rotary(q, k, p, rotary, backward=back)
                for got, x in ((a, q), (b, k)):
                    want = R.rotate(x.transpose(0, 1), p, rotary.inv_freq, rotary.magnitude, interleaved, back).transpose(0, 1)
                    _rot_close(got, want, x)
                    assert torch.equal(got[..., rot:], x[..., rot:])
        alone = S.sage_rotary(q, None, pos, rotary)
        assert torch.equal(alone, S.sage_rotary(q, k, pos, rotary)[0])


@pytest.mark.parametrize("layout", ["HND", "NHD"])
def test_rotary_layouts_views_and_in_place(layout):
    b, n, d = 3, 29, 128
    rotary = S.SageRotary(d, rotary_dim=64)
    qkv = torch.randn((b, n, 3, 4, d), device="cuda").half()
    q, k = qkv[:, :, 0], qkv[:, :, 1]
    if layout == "HND":
        q, k = q.transpose(1, 2), k.transpose(1, 2)
    pos = torch.randint(0, 5000, (b, n), device="cuda")
    a, c = S.sage_rotary(q, k, pos, rotary, tensor_layout=layout)
    for i in range(b):
        x = qkv[i, :, 0]
        want = S.sage_rotary(x, None, pos[i], rotary)
        assert torch.equal(a[i] if layout == "NHD" else a[i].transpose(0, 1), want)
    same = S.sage_rotary(q, k, pos[0], rotary, tensor_layout=layout)[0]
    assert torch.equal(same[0], a[0])
    rest = qkv[:, :, 2].clone()
    got = S.sage_rotary(q, k, pos, rotary, tensor_layout=layout, out=(q, k))
    assert got[0].data_ptr() == q.data_ptr() and torch.equal(q, a) and torch.equal(k, c) and torch.equal(qkv[:, :, 2], rest)


def test_rotary_gradient():
    """Against the formula, against differences, and that the transposed map of the map is the length squared."""
    n, d = 11, 64
    rotary = S.SageRotary(d, rotary_dim=48, scaling="parts", factor=8.0)
    q = torch.randn((n, 3, d), device="cuda").half().requires_grad_()
    k = torch.randn((n, 1, d), device="cuda").half().requires_grad_()
    pos = torch.arange(n, device="cuda") * 1000
    a, b = S.sage_rotary(q, k, pos, rotary)
    ga, gb = torch.randn_like(a), torch.randn_like(b)
    torch.autograd.backward((a, b), (ga, gb))
    for x, g in ((q, ga), (k, gb)):
        want = R.rotate(g.transpose(0, 1), pos, rotary.inv_freq, rotary.magnitude, False, True).transpose(0, 1)
        _rot_close(x.grad, want, g)
    # one gradient only, broadcast gradients
    x = torch.randn((n, 2, d), device="cuda").half().requires_grad_()
    S.sage_rotary(x, None, pos, rotary).sum().backward()
    want = R.rotate(torch.ones((2, n, d), device="cuda"), pos, rotary.inv_freq, rotary.magnitude, False, True).transpose(0, 1)
    _rot_close(x.grad, want, torch.ones_like(x))
    # differences: the map is linear, so a step of any size does; <g, R(x + e) - R(x)> = <R^T g, e>
    with torch.no_grad():
        e = torch.randn_like(q)
        y = S.sage_rotary(q, None, pos, rotary).double()
        y2 = S.sage_rotary((q + e).half(), None, pos, rotary).double()
        step = (q + e).half().double() - q.double()
        lhs, rhs = ((y2 - y) * ga.double()).sum(), (q.grad.double() * step).sum()
        # three fp16 roundings of values of up to about 6 x 1.21, over n x 3 x d terms that add like a random walk
        assert abs(lhs - rhs) <= 6 * (n * 3 * d) ** 0.5 * 3 * 8 * 2.0 ** -11
    # a pass backwards that is captured while an eager graph of the same leaf lives
    eager = S.sage_rotary(q, None, pos, rotary)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    g = torch.ones_like(eager)
    with torch.no_grad(), torch.cuda.stream(st):
        S.sage_rotary(g, None, pos, rotary, backward=True)
        st.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=st):
            back = S.sage_rotary(g, None, pos, rotary, backward=True)
    gr.replay()
    torch.cuda.synchronize()
    (grad,) = torch.autograd.grad(eager, q, g)
    assert torch.equal(back, grad)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_generation_step_by_step(dtype):
    """As a program uses them: a prompt rotated and written, then tokens one at a time, then a drafted chain verified at
    once, against the same attention over the same cache for all positions in 64 bits; and the cache read back for
    `sageattn_varlen`."""
    dt, hq, hkv, d, page, prompt, steps = DT[dtype], 8, 2, 128, 16, 45, 6
    n = prompt + steps
    rotary = S.SageRotary(d, scaling="ntk", factor=2.0)
    cache = S.SageCache.empty(6, page, hkv, d, dtype=dt)
    table = torch.tensor([[4, 1, 5, 0]], dtype=torch.int32, device="cuda")
    q, k, v = (torch.randn((n, h, d), device="cuda").to(dt) for h in (hq, hkv, hkv))
    pos = torch.arange(n, device="cuda")
    slots = table[0, pos // page].long() * page + pos % page
    qr, kr = S.sage_rotary(q, k, pos, rotary)
    S.sage_cache_write(cache, kr[:prompt], v[:prompt], slots[:prompt])
    lens = torch.tensor([prompt], dtype=torch.int32, device="cuda")
    outs = [S.sageattn_cached(qr[:prompt], cache, table, lens)]
    for i in range(prompt, n):
        q1, k1 = S.sage_rotary(q[i:i + 1], k[i:i + 1], pos[i:i + 1], rotary)
        assert torch.equal(q1[0], qr[i]) and torch.equal(k1[0], kr[i])
        S.sage_cache_write(cache, k1, v[i:i + 1], slots[i:i + 1])
        lens += 1
        outs.append(S.sageattn_cached(q1, cache, table, lens))
    out = torch.cat(outs)
    want, _ = R.attend_cached(qr, cache, table, [n], [0, n])
    top = R.values(cache.v_codes, cache.v_scale, table[0], n, d)[0].abs().max()
    bound = 1.25 * 2.0 ** -11 * top + torch.finfo(dt).eps / 2 * want.abs()
    assert ((out.double() - want).abs() <= bound).all()
    chain = S.sageattn_cached(qr[prompt:], cache, table, lens, tree_mask=torch.ones((steps, steps), device="cuda").tril().bool())
    assert ((chain.double() - want[prompt:]).abs() <= bound[prompt:]).all()
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    k16, v16 = S.sage_cache_read(cache, table, cu, n, dtype=dt)
    full = S.sageattn_varlen(qr, k16, v16, cu, cu, n, n, is_causal=True)
    be.check()
    # sageattn quantises Q and P too: e4m3 weights are off by 2^-4 each, of which a row's sum keeps a random walk
    assert (full.double() - want).norm() / want.norm() < 0.05
