"""What the Python layer of the cache operators refuses on the GPU, before anything is launched."""
import pytest
import torch

import sageattention as S

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def setup():
    cache = S.SageCache.empty(4, 16, 2, 64)
    x = torch.zeros((3, 2, 64), dtype=torch.float16, device="cuda")
    q = torch.zeros((3, 4, 64), dtype=torch.float16, device="cuda")
    return cache, x, q, torch.zeros((3, 2), dtype=torch.int32, device="cuda"), torch.ones(3, dtype=torch.int32, device="cuda")


def test_write(setup):
    cache, x, _, _, _ = setup
    slots = torch.arange(3, device="cuda")
    for args in ((x.cpu(), x, slots), (x, x, slots.cpu()), (x.float(), x.float(), slots), (x, x.bfloat16(), slots), (x[:2], x, slots), (x, x, slots[:2]),
                 (x, x, slots.float()), (x[:, :1], x[:, :1], slots), (x[..., :32], x[..., :32], slots), (x.unsqueeze(0), x.unsqueeze(0), slots),
                 (x.transpose(1, 2).contiguous().transpose(1, 2), x, slots), (x, x, torch.zeros(6, dtype=torch.int64, device="cuda")[::2])):
        with pytest.raises(ValueError):
            S.sage_cache_write(cache, *args)


def test_read(setup):
    cache, x, _, table, _ = setup
    cu = torch.arange(4, dtype=torch.int32, device="cuda")
    ok = (table, cu, 3)
    S.sage_cache_read(cache, *ok)
    for args, kw in (((table.cpu(), cu, 3), {}), ((table.long(), cu, 3), {}), ((table, cu.long(), 3), {}), ((table, cu[:3], 3), {}), ((table[0], cu, 3), {}),
                     ((table, cu, -1), {}), (ok, dict(dtype=torch.float32)), (ok, dict(out=(x[:2], x))), (ok, dict(out=(x, x.bfloat16()))),
                     ((table[:, :0], cu, 3), {}), ((table.T.contiguous().T, cu, 3), {})):
        with pytest.raises(ValueError):
            S.sage_cache_read(cache, *args, **kw)


def test_attention(setup):
    cache, _, q, table, lens = setup
    cu = torch.arange(4, dtype=torch.int32, device="cuda")
    tree = torch.ones((3, 1), dtype=torch.bool, device="cuda")
    S.sageattn_cached(q, cache, table, lens, cu, 1, tree_mask=tree)
    assert S.sageattn_cached(q[:0], cache, table, lens).shape == (0, 4, 64)
    for args, kw in (((q.cpu(), cache, table, lens), {}), ((q.float(), cache, table, lens), {}), ((q[:, :3], cache, table, lens), {}),
                     ((q[..., :32], cache, table, lens), {}), ((q, cache, table.long(), lens), {}), ((q, cache, table, lens.long()), {}),
                     ((q, cache, table, lens[:2]), {}), ((q[:2], cache, table, lens), {}), ((q, cache, table, lens), dict(max_seqlen_q=2)),
                     ((q, cache, table, lens, cu), {}), ((q, cache, table, lens, cu, 0), {}), ((q, cache, table, lens, cu[:3], 1), {}),
                     ((q, cache, table, lens, cu.long(), 1), {}), ((q, cache, table, lens, cu, 2), dict(tree_mask=tree)),
                     ((q, cache, table, lens), dict(tree_mask=tree.float())), ((q, cache, table, lens), dict(tree_mask=tree[:2])),
                     ((q, cache, table, lens), dict(sm_scale=0.0)), ((q, cache, table, lens), dict(sm_scale=float("nan"))),
                     ((q, cache, table, lens), dict(out=q[:2])), ((q, cache, table, lens), dict(out=q.bfloat16())),
                     ((q.transpose(1, 2).contiguous().transpose(1, 2), cache, table, lens), {}), ((q, cache, table.cpu(), lens), {})):
        with pytest.raises(ValueError):
            S.sageattn_cached(*args, **kw)


def test_rotary(setup):
    _, k, q, _, _ = setup
    rotary, pos = S.SageRotary(64), torch.arange(3, device="cuda")
    S.sage_rotary(q, k, pos, rotary)
    grad = q.clone().requires_grad_()
    wide = torch.zeros((3, 4, 128), dtype=torch.float16, device="cuda")
    for args, kw in (((q, k, pos.cpu(), rotary), {}), ((q, k, pos.float(), rotary), {}), ((q, k, pos[:2], rotary), {}), ((q, k[:2], pos, rotary), {}),
                     ((q, k.bfloat16(), pos, rotary), {}), ((q, k, pos, S.SageRotary(128)), {}), ((q[0], None, pos, rotary), {}),
                     ((q, k, pos, rotary), dict(tensor_layout="BSHD")), ((grad, k, pos, rotary), dict(out=(q, k))), ((q, k, pos, rotary), dict(out=q)),
                     ((q, k, pos, rotary), dict(out=(q[:2], k))), ((wide[..., :64], None, pos, rotary), dict(out=wide[..., 32:96])),
                     ((q, k, pos, S.SageRotary(64, device="cpu")), {}), ((q, k, pos[None], rotary), {})):
        with pytest.raises(ValueError):
            S.sage_rotary(*args, **kw)


def test_outputs_that_share_memory(setup):
    cache, x, q, table, lens = setup
    cu = torch.arange(4, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        S.sageattn_cached(q, cache, table, lens, out=q)
    both = torch.zeros((6, 4, 64), dtype=torch.float16, device="cuda")
    with pytest.raises(ValueError):
        S.sageattn_cached(both[:3], cache, table, lens, out=both[2:5])
    S.sageattn_cached(both[:3], cache, table, lens, out=both[3:])
    with pytest.raises(ValueError):
        S.sage_cache_read(cache, table, cu, 3, out=(x, x))
    fused = torch.zeros((3, 4, 64), dtype=torch.float16, device="cuda")
    S.sage_cache_read(cache, table, cu, 3, out=(fused[:, :2], fused[:, 2:]))


def test_buffers_are_fixed(setup):
    cache = setup[0]
    for name in ("k_codes", "v_codes", "k_scale", "v_scale", "k_shift", "num_pages"):
        with pytest.raises(AttributeError):
            setattr(cache, name, getattr(cache, name))


def test_autograd_learns_of_outputs(setup):
    cache, _, q, table, lens = setup
    w = q.clone().requires_grad_()
    held = q.clone()
    y = (w * held).sum()                             # keeps `held` for its backward pass
    S.sage_rotary(held, None, torch.arange(3, device="cuda"), S.SageRotary(64), out=held)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_nothing_to_do(setup):
    cache, x, q, table, lens = setup
    k, v = S.sage_cache_read(cache, table, torch.zeros(4, dtype=torch.int32, device="cuda"), 0)
    assert k.shape == v.shape == (0, 2, 64) and k.dtype == torch.float16
    out, lse = S.sageattn_cached(q[:0], cache, table, lens, return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4) and lse.dtype == torch.float32
    S.sage_cache_write(cache, x[:0], x[:0], torch.zeros(0, dtype=torch.int64, device="cuda"))
    assert S.sage_rotary(q[:0], None, torch.zeros(0, dtype=torch.int64, device="cuda"), S.SageRotary(64)).shape == (0, 4, 64)
