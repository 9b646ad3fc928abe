"""What the cache operators refuse, and their host side, without a GPU: every call below must stop at validation."""
import ctypes
import math

import pytest
import torch

import sageattention as S
from sageattention import _native, cache as C

buf = (ctypes.c_char * 4096)()
P = (ctypes.addressof(buf) + 255) // 256 * 256
S2, S3 = _native.strides2(1024, 128), _native.strides3(8192, 1024, 128)
ARG, UNSUPPORTED, WORKSPACE = _native.SAGE_E_ARG, _native.SAGE_E_UNSUPPORTED, _native.SAGE_E_WORKSPACE


def _refused(rc, code, word):
    assert rc == code, (rc, _native.load().sage_last_error())
    assert word.encode() in _native.load().sage_last_error(), _native.load().sage_last_error()


def _write(k=P, v=P, slots=P, s64=1, kc=P, ks=P, vc=P, vs=P, shift=None, tokens=4, heads=8, d=128, pages=4, page=64,
           k_st=S2, v_st=S2, dtype=0, mode=0):
    return _native.load().sage_cache_write(k, v, slots, s64, kc, ks, vc, vs, shift, tokens, heads, d, pages, page, k_st, v_st, dtype, mode, None)


def _read(kc=P, table=P, stride=4, width=4, cu=P, k=P, v=P, n_seq=1, total=4, heads=8, d=128, pages=4, page=64, k_st=S2, v_st=S2, dtype=0, mode=0):
    return _native.load().sage_cache_read(kc, P, P, P, None, table, stride, width, cu, k, v, n_seq, total, heads, d, pages, page, k_st, v_st, dtype, mode, None)


def _attend(q=P, out=P, lse=None, kc=P, table=P, stride=4, width=4, lens=P, cu=P, tree=None, tree_st=0, ws=P, ws_bytes=1 << 40, n_seq=1,
            hq=8, hkv=8, total=4, max_q=4, d=128, pages=4, page=64, q_st=S2, o_st=S2, dtype=0, mode=0, scale=0.1, status=None):
    return _native.load().sage_cache_attention(q, out, lse, kc, P, P, P, None, table, stride, width, lens, cu, tree, tree_st, ws, ws_bytes,
                                               n_seq, hq, hkv, total, max_q, d, pages, page, q_st, o_st, dtype, mode, scale, status, None)


def _rotary(q=P, qo=P, k=None, ko=None, pos=P, p64=1, freq=P, b=1, hq=8, hk=0, n=4, d=128, rot=128, st=S3, p2=_native.strides2(0, 1), dtype=0):
    return _native.load().sage_rotary(q, qo, k, ko, pos, p64, freq, 1.0, b, hq, hk, n, d, rot, 0, 0, st, S3, S3, S3, p2, dtype, None)


@pytest.mark.parametrize("call", [_write, _read, _attend])
def test_cache_shapes(call):
    for d in (0, 4, 12, 136):
        _refused(call(d=d), UNSUPPORTED, "head_dim")
    for page in (0, 8, 24, 512, -16):
        _refused(call(page=page), UNSUPPORTED, "page_size")
    _refused(call(pages=0), ARG, "pages")
    _refused(call(pages=1 << 31), ARG, "pages")
    _refused(call(dtype=2), ARG, "dtype")
    _refused(call(mode=2), ARG, "qk_mode")
    _refused(call(kc=None), ARG, "null")
    _refused(call(kc=P + 8), ARG, "aligned")


def test_write_refusals():
    assert _write(tokens=0) == 0
    for name in ("k", "v", "slots"):
        _refused(_write(**{name: None}), ARG, "null")
    _refused(_write(tokens=-1), ARG, "token")
    _refused(_write(heads=0), ARG, "heads")
    _refused(_write(k=P + 2), ARG, "aligned")
    _refused(_write(slots=P + 4), ARG, "slots")
    _refused(_write(slots=P + 2, s64=0), ARG, "slots")
    for bad in ((0, 128), (1024, -8), (1020, 128)):
        _refused(_write(v_st=_native.strides2(*bad)), ARG, "stride")
    _refused(_write(k_st=_native.strides2(1 << 39, 128)), UNSUPPORTED, "2^39")
    _refused(_write(k_st=None), ARG, "strides")


def test_read_refusals():
    assert _read(total=0) == 0
    for name in ("cu", "k", "v", "table"):
        _refused(_read(**{name: None}), ARG, "null")
    _refused(_read(n_seq=0), ARG, "sequences")
    _refused(_read(n_seq=65536), ARG, "sequences")
    _refused(_read(width=0), ARG, "width")
    _refused(_read(stride=-1), ARG, "stride")
    _refused(_read(width=1 << 28), UNSUPPORTED, "2^30")
    _refused(_read(total=-1), ARG, "row count")
    _refused(_read(cu=P + 2), ARG, "aligned")
    _refused(_read(k=P + 8), ARG, "aligned")


def test_attention_refusals():
    assert _attend(total=0) == 0
    for name in ("q", "out", "lens", "table", "ws"):
        _refused(_attend(**{name: None}), ARG, "null")
    _refused(_attend(cu=None, n_seq=3), ARG, "max_q")
    _refused(_attend(hq=9), ARG, "multiple")
    _refused(_attend(hq=0), ARG, "heads")
    _refused(_attend(max_q=0), ARG, "max_q")
    _refused(_attend(max_q=5), ARG, "max_q")
    _refused(_attend(lse=P + 2), ARG, "aligned")
    _refused(_attend(q=P + 8), ARG, "aligned")
    _refused(_attend(status=P + 2), ARG, "status_host")
    _refused(_attend(tree=P, tree_st=-1), ARG, "tree_stride")
    _refused(_attend(ws=P + 16), ARG, "256")
    _refused(_attend(ws_bytes=100), WORKSPACE, "needs")
    for scale in (0.0, -1.0, math.inf, math.nan):
        _refused(_attend(scale=scale), ARG, "sm_scale")
    _refused(_attend(total=1 << 30, max_q=1 << 30), UNSUPPORTED, "rows")
    lib = _native.load()
    assert lib.sage_cache_attention_workspace_bytes(1, 8, 3, 1) == 0 and lib.sage_cache_attention_workspace_bytes(0, 8, 8, 1) == 0
    assert lib.sage_cache_attention_workspace_bytes(4, 8, 8, 1) % 256 == 0


def test_rotary_refusals():
    assert _rotary(n=0) == 0 and _rotary(b=0) == 0
    for name in ("q", "qo", "pos", "freq"):
        _refused(_rotary(**{name: None}), ARG, "null")
    _refused(_rotary(k=P, ko=None, hk=2), ARG, "null")
    for rot in (0, 4, 12, 136):
        _refused(_rotary(rot=rot), UNSUPPORTED, "rotary_dim")
    _refused(_rotary(d=64, rot=72), UNSUPPORTED, "rotary_dim")
    _refused(_rotary(d=12), UNSUPPORTED, "head_dim")
    _refused(_rotary(hq=0), ARG, "sizes")
    _refused(_rotary(dtype=3), ARG, "dtype")
    _refused(_rotary(pos=P + 4), ARG, "misaligned")
    _refused(_rotary(freq=P + 4), ARG, "misaligned")
    _refused(_rotary(q=P + 8), ARG, "aligned")
    _refused(_rotary(p2=_native.strides2(-1, 1)), ARG, "position stride")
    _refused(_rotary(st=_native.strides3(8, 8, 4)), ARG, "stride")
    _refused(_rotary(n=1 << 31), UNSUPPORTED, "tokens")


def test_python_layer_has_no_cpu_path():
    codes, scale = torch.zeros((2, 1, 16, 128), dtype=torch.int8), torch.zeros((2, 1, 16))
    with pytest.raises(ValueError, match="CUDA"):
        S.SageCache(codes, scale, codes.view(torch.float8_e4m3fn), scale, 128)
    with pytest.raises(ValueError, match="CUDA"):
        S.SageCache.empty(2, 16, 1, 128, device="cpu")
    rotary = S.SageRotary(64, device="cpu")
    x = torch.zeros((2, 3, 64), dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        S.sage_rotary(x, None, torch.zeros(2, dtype=torch.int32), rotary)


def test_cache_buffers_are_checked():
    codes, scale = torch.zeros((2, 1, 16, 128), dtype=torch.int8), torch.zeros((2, 1, 16))
    e4m3 = codes.view(torch.float8_e4m3fn)
    for args, kind, word in (((codes[0], scale, e4m3, scale, 128), ValueError, "k_codes"), ((codes.view(torch.uint8), scale, e4m3, scale, 128), ValueError, "k_codes"),
                             ((codes, scale, codes, scale, 128), ValueError, "v_codes"), ((codes, scale[:1], e4m3, scale, 128), ValueError, "k_scale"),
                             ((codes, scale, e4m3, scale.half(), 128), ValueError, "v_scale"), ((codes, scale, e4m3, scale, 64), ValueError, "64 bytes"),
                             ((codes, scale, e4m3, scale, 12), NotImplementedError, "head_dim"),
                             ((codes[:, :, :8], scale[:, :, :8], e4m3[:, :, :8], scale[:, :, :8], 128), NotImplementedError, "page_size")):
        with pytest.raises(kind, match=word):
            S.SageCache(*args)


def test_rotary_frequencies():
    base = [10000.0 ** (-i / 64) for i in range(0, 64, 2)]
    assert S.SageRotary(128, rotary_dim=64, device="cpu").inv_freq.tolist() == base
    linear = S.SageRotary(64, scaling="linear", factor=4.0, device="cpu")
    assert linear.inv_freq.tolist() == [f / 4 for f in base] and linear.magnitude == 1.0
    ntk = S.SageRotary(64, scaling="ntk", factor=4.0, device="cpu").inv_freq
    # the slowest pair turns `factor` times as slowly, the fastest as before
    assert ntk[0] == 1.0 and abs(ntk[-1].item() * 4 / base[-1] - 1) < 1e-12
    parts = S.SageRotary(64, scaling="parts", factor=4.0, original_length=4096, device="cpu")
    turns = [4096 * f / (2 * math.pi) for f in base]
    for f, t, got in zip(base, turns, parts.inv_freq.tolist()):
        if t >= 32:
            assert got == f
        elif t <= 1:
            assert got == f / 4
        else:
            assert f / 4 < got < f
    assert abs(parts.magnitude - (0.1 * math.log(4) + 1)) < 1e-15
    for kw, kind in ((dict(rotary_dim=12), NotImplementedError), (dict(rotary_dim=72), NotImplementedError), (dict(scaling="cubic"), ValueError),
                     (dict(factor=0.5), ValueError), (dict(base=1.0), ValueError), (dict(scaling="parts", slow=0.0), ValueError)):
        with pytest.raises(kind):
            S.SageRotary(64, device="cpu", **kw)


def test_shared_elements_of_views():
    """The exact test for views with the same strides against an enumeration of their elements."""
    gen = torch.Generator().manual_seed(0)
    store = torch.zeros(4096, dtype=torch.float16)

    def elements(t):
        at = [t.data_ptr() // 2]
        for n, s in zip(t.shape, t.stride()):
            at = [x + i * s for x in at for i in range(n)]
        return set(at)

    seen = set()
    for _ in range(400):
        full = torch.randint(1, 5, (4,), generator=gen).tolist()
        strides = [full[1] * full[2] * full[3], full[2] * full[3], full[3], 1]
        a, b = (store.as_strided([int(torch.randint(1, n + 1, (1,), generator=gen)) for n in full], strides, int(torch.randint(0, 200, (1,), generator=gen)))
                for _ in range(2))
        want = bool(elements(a) & elements(b))
        assert C._overlap(a, b) == want
        seen.add(want)
    assert seen == {True, False}
    assert C._overlap(store[:64].view(8, 8), store[32:96].view(8, 8).T) and not C._overlap(store[:64].view(8, 8), store[64:128].view(4, 16))


def test_buffers_and_frequencies_are_fixed():
    rotary = S.SageRotary(64, device="cpu")
    for name, value in (("inv_freq", torch.zeros(4, dtype=torch.float64)), ("magnitude", 2.0), ("rotary_dim", 128)):
        with pytest.raises(AttributeError):
            setattr(rotary, name, value)
    assert rotary.magnitude == 1.0 and rotary.rotary_dim == 64


def test_calls_in_words():
    """Argument by argument, the words reach the same checks."""
    import struct
    lib = _native.load()
    code = (ctypes.addressof(buf) + 255) // 256 * 256
    two = (1024, 128)
    write = [code] * 3 + [0] + [1] + [code] * 5 + [4, 8, 128, 4, 64, *two, *two, 0, 0]
    read = [code] * 4 + [0] + [code] * 5 + [4, 4, 1, 4, 8, 128, 4, 64, *two, *two, 0, 0]
    attend = [code] * 8 + [1 << 40, 0, 0] + [code] * 5 + [4, 4, 4, 1, 8, 8, 4, 4, 128, 4, 64, *two, *two, 0, 0, 0.1]
    rotary = [code] * 5 + [0, 0] + [code, 1, 1.0, 1, 8, 8, 4, 128, 128, 0] + [8192, 1024, 128] * 4 + [0, 1, 0]

    def call(what, words, change=(), count=None):
        words = list(words)
        for i, x in change:
            words[i] = x
        data = struct.pack("".join("d" if isinstance(x, float) else "q" for x in words), *words)
        return lib.sage_call_words(what, data, len(words) if count is None else count)

    for what, words in enumerate((write, read, attend, rotary)):
        assert len(words) == C._COUNT[what]
        _refused(call(what, words[:-1]), ARG, "words")
        _refused(call(what, words + [0]), ARG, "words")
        _refused(call(what, words, [(0, code + 2)]), ARG, "aligned")
    _refused(call(4, write), ARG, "words")
    _refused(call(-1, write), ARG, "words")
    _refused(lib.sage_call_words(0, None, 21), ARG, "words")
    for at, value, rc, word in ((12, 136, UNSUPPORTED, "head_dim"), (13, 0, ARG, "pages"), (14, 24, UNSUPPORTED, "page_size"), (19, 2, ARG, "dtype"),
                                (20, 2, ARG, "qk_mode"), (15, 4, ARG, "stride"), (18, 4, ARG, "stride"), (10, -1, ARG, "token")):
        _refused(call(0, write, [(at, value)]), rc, word)
    for at, value, rc, word in ((15, 136, UNSUPPORTED, "head_dim"), (16, 0, ARG, "pages"), (17, 24, UNSUPPORTED, "page_size"), (22, 2, ARG, "dtype"),
                                (23, 2, ARG, "qk_mode"), (18, 4, ARG, "stride"), (21, 4, ARG, "stride"), (13, -1, ARG, "row"), (11, 0, ARG, "table")):
        _refused(call(1, read, [(at, value)]), rc, word)
    for at, value, rc, word in ((24, 136, UNSUPPORTED, "head_dim"), (25, 0, ARG, "pages"), (26, 24, UNSUPPORTED, "page_size"), (31, 2, ARG, "dtype"),
                                (32, 2, ARG, "qk_mode"), (27, 4, ARG, "stride"), (30, 4, ARG, "stride"), (22, -1, ARG, "token"), (17, 0, ARG, "table"),
                                (33, -1.0, ARG, "sm_scale"), (8, 16, WORKSPACE, "workspace"), (18, -1, ARG, "tree"), (20, 9, ARG, "heads"),
                                (23, 5, ARG, "max_q"), (9, code + 2, ARG, "status_host"), (4, 0, ARG, "null")):
        _refused(call(2, attend, [(at, value)]), rc, word)
    for at, value, rc, word in ((14, 136, UNSUPPORTED, "head_dim"), (15, 4, UNSUPPORTED, "rotary_dim"), (31, 2, ARG, "dtype"), (17, 4, ARG, "stride"),
                                (28, 4, ARG, "stride"), (29, -1, ARG, "position"), (10, -1, ARG, "sizes"), (7, code + 4, ARG, "misaligned")):
        _refused(call(3, rotary, [(at, value)]), rc, word)


def test_copies_have_frequencies_of_their_own():
    import copy
    import pickle
    rotary = S.SageRotary(96, rotary_dim=64, interleaved=True, scaling="parts", factor=4.0, device="cpu")
    rotary._plans["call"] = b"addresses"
    for twin in (copy.deepcopy(rotary), pickle.loads(pickle.dumps(rotary)), copy.copy(rotary)):
        assert not twin._plans and twin.inv_freq.device == rotary.inv_freq.device and torch.equal(twin.inv_freq, rotary.inv_freq)
        assert (twin.head_dim, twin.rotary_dim, twin.interleaved, twin.magnitude) == (96, 64, True, rotary.magnitude)
    assert copy.deepcopy(rotary).inv_freq.data_ptr() != rotary.inv_freq.data_ptr()


def _recorded(monkeypatch):
    """The Python layer on CPU tensors: a plan is its output's strides in words, a C call is recorded instead of made."""
    calls = []
    monkeypatch.setattr(C, "_raw_stream", lambda index: 0)
    monkeypatch.setattr(C, "_call", lambda what, dev, words: calls.append(words) or 0)
    monkeypatch.setattr(C, "_plan_rotary", lambda q, k, positions, rotary, layout, out: b"fresh" if out is None else b"given")
    return calls


@pytest.mark.parametrize("fresh_first", [True, False])
def test_fresh_and_in_place_rotations_have_plans_of_their_own(monkeypatch, fresh_first):
    calls = _recorded(monkeypatch)
    rotary, pos = S.SageRotary(64, device="cpu"), torch.arange(5)
    q = torch.zeros((5, 6, 64), dtype=torch.float16)[:, :2]          # strided, as a part of a fused projection
    for _ in range(2):
        for fresh in (fresh_first, not fresh_first):
            C._rotate(q, None, pos, rotary, "HND", False, None if fresh else q)
            assert calls.pop().endswith(b"fresh" if fresh else b"given")
    # one tensor as both inputs: the outputs of a call in place would overlap, which only its own checks can see
    for fresh in (fresh_first, not fresh_first):
        C._rotate(q, q, pos, rotary, "HND", False, None if fresh else (q, q))
        assert calls.pop().endswith(b"fresh" if fresh else b"given")


@pytest.mark.parametrize("layout", ["HND", "NHD"])
def test_rotary_refuses_a_packed_tensor_next_to_a_batched_one(layout):
    rotary, pos = S.SageRotary(64, device="cpu"), torch.arange(5)
    packed = torch.zeros((5, 2, 64), dtype=torch.float16)
    batched = torch.zeros((1, 5, 2, 64) if layout == "NHD" else (1, 2, 5, 64), dtype=torch.float16)
    for q, k in ((packed, batched), (batched, packed)):
        with pytest.raises(ValueError, match="both"):
            S.sage_rotary(q, k, pos, rotary, tensor_layout=layout)


def test_shared_elements_of_views_with_axes_of_one():
    """As above with axes of one element at any stride, 0 among them, and with axes that lie over each other."""
    gen = torch.Generator().manual_seed(1)
    store = torch.zeros(4096, dtype=torch.float16)
    pick = lambda lo, hi: int(torch.randint(lo, hi, (1,), generator=gen))

    def elements(t):
        at = [t.data_ptr() // 2]
        for n, s in zip(t.shape, t.stride()):
            at = [x + i * s for x in at for i in range(n)]
        return set(at)

    seen = set()
    for _ in range(600):
        ones = [pick(0, 2) for _ in range(3)]
        full = [1 if one else pick(2, 5) for one in ones] + [pick(1, 9)]
        strides, step = [0, 0, 0, 1], full[3]
        for i in (2, 1, 0):
            strides[i] = pick(0, 60) if ones[i] else step
            step *= full[i]
        a, b = (store.as_strided([n if one else pick(1, n + 1) for n, one in zip(full, ones + [0])], strides, pick(0, 100)) for _ in range(2))
        want = bool(elements(a) & elements(b))
        assert C._overlap(a, b) == want, (a.shape, b.shape, strides)
        seen.add(want)
    assert seen == {True, False}
    # what cannot be told apart exactly counts as sharing: never a miss
    for _ in range(300):
        strides = [pick(0, 9) for _ in range(3)]
        a, b = (store.as_strided([pick(1, 4) for _ in range(3)], strides, pick(0, 20)) for _ in range(2))
        assert C._overlap(a, b) or not elements(a) & elements(b), (a.shape, b.shape, strides)


def _host_cache(pages=4, page=16, heads=2, d=64):
    """What the checks of a call read of a cache, on the CPU."""
    from types import SimpleNamespace
    return SimpleNamespace(device=torch.device("cpu"), num_kv_heads=heads, head_dim=d, _sizes=(pages, page), _args=(0,) * 5, _mode=0, num_pages=pages,
                           page_size=page, _plans={})


def test_rows_of_an_output_have_memory_of_their_own():
    cache, store = _host_cache(), torch.zeros(4096, dtype=torch.float16)
    table, lens, cu = torch.zeros((3, 2), dtype=torch.int32), torch.ones(3, dtype=torch.int32), torch.arange(4, dtype=torch.int32)
    q, x = torch.zeros((3, 4, 64), dtype=torch.float16), torch.zeros((3, 2, 64), dtype=torch.float16)
    view = lambda shape, *strides: store.as_strided(shape, (*strides, 1))
    for strides in ((256, 64), (64, 192), (512, 72), (72, 512)):     # rows side by side, tokens or heads first
        C._plan_attend(cache, q, table, lens, None, None, None, None, view((3, 4, 64), *strides))
        C._plan_read(cache, table, cu, 3, torch.float16, (view((3, 2, 64), *strides), x))
    for strides in ((64, 64), (8, 64), (256, 8), (128, 64), (64, 128)):
        with pytest.raises(ValueError, match="overlap"):
            C._plan_attend(cache, q, table, lens, None, None, None, None, view((3, 4, 64), *strides))
    for strides in ((64, 64), (8, 128), (128, 8), (64, 128)):
        with pytest.raises(ValueError, match="overlap"):
            C._plan_read(cache, table, cu, 3, torch.float16, (view((3, 2, 64), *strides), x))
    one = C._plan_attend(cache, q[:1], table[:1], lens[:1], None, None, None, None, view((1, 4, 64), 8, 64))     # a single token has no next one
    assert one[0]
    same = C._plan_attend(cache, view((3, 4, 64), 8, 8), table, lens, None, None, None, None, None)             # inputs may
    assert same[0]


def test_rotary_refuses_forward_mode_derivatives(monkeypatch):
    import torch.autograd.forward_ad as fw
    calls = _recorded(monkeypatch)
    rotary, pos, x = S.SageRotary(64, device="cpu"), torch.arange(5), torch.zeros((5, 2, 64), dtype=torch.float16)
    with fw.dual_level():
        dual = fw.make_dual(x, torch.ones_like(x))
        for args in ((dual, None), (dual, x), (x, dual)):
            with pytest.raises(NotImplementedError):
                S.sage_rotary(*args, pos, rotary)
        with torch.no_grad(), pytest.raises(NotImplementedError):
            S.sage_rotary(dual, None, pos, rotary)
        with pytest.raises(NotImplementedError):
            S.sage_rotary(fw.make_dual(x.clone().requires_grad_(), torch.ones_like(x)), None, pos, rotary)
        assert not calls
        S.sage_rotary(x, x, pos, rotary)             # the level alone changes nothing
    assert len(calls) == 1


def test_outputs_that_require_gradients_are_refused(monkeypatch):
    calls = _recorded(monkeypatch)
    rotary, pos = S.SageRotary(64, device="cpu"), torch.arange(5)
    x, leaf = torch.zeros((5, 2, 64), dtype=torch.float16), torch.zeros((5, 2, 64), dtype=torch.float16, requires_grad=True)
    later = leaf * 2
    for out in (leaf, later):
        with pytest.raises(ValueError, match="gradients"):
            S.sage_rotary(x, None, pos, rotary, out=out)
        with pytest.raises(ValueError, match="gradients"):
            S.sage_rotary(x, x.clone(), pos, rotary, out=(torch.zeros_like(x), out))
    table, cu = torch.zeros((1, 1), dtype=torch.int32), torch.tensor([0, 5], dtype=torch.int32)
    with pytest.raises(ValueError, match="gradients"):
        S.sage_cache_read(_host_cache(), table, cu, 5, out=(x, leaf))
    assert not calls
    with torch.no_grad():                            # a parameter may be turned in place, as it may be written to
        S.sage_rotary(leaf, None, pos, rotary, out=leaf)
    assert len(calls) == 1


def test_autograd_learns_of_writes_to_the_cache(monkeypatch):
    calls = _recorded(monkeypatch)
    cache = _host_cache()
    cache._tracked = [torch.ones(4), torch.ones(4)]
    w = torch.ones(4, requires_grad=True)
    y = (w * cache._tracked[1]).sum()                # keeps the scales for its backward pass
    x = torch.zeros((3, 2, 64), dtype=torch.float16)
    S.sage_cache_write(cache, x, x, torch.arange(3))
    assert len(calls) == 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_gradients_arrive_as_the_kernel_takes_them(monkeypatch):
    """Broadcast, at an odd offset of a larger gradient, with an axis of one of any stride."""
    _recorded(monkeypatch)
    taken = []

    def plan(q, k, positions, rotary, layout, out):
        taken.extend(C.strided_view_reason(C._rotary_views(x, layout)) for x in (q, k) if x is not None)
        return b""
    monkeypatch.setattr(C, "_plan_rotary", plan)
    monkeypatch.setattr(C, "_remember", lambda plans, key, words: words)
    rotary = S.SageRotary(64, device="cpu")
    for n in (1, 5):
        pos = torch.arange(n)
        q = torch.zeros((n, 2, 64), dtype=torch.float16, requires_grad=True)
        odd = torch.zeros(3, dtype=torch.float16, requires_grad=True)
        a, b = S.sage_rotary(q, q, pos, rotary)
        torch.cat([odd, a.flatten(), b.flatten()]).pow(2).sum().backward()
        S.sage_rotary(q, None, pos, rotary).sum().backward()
        strange = torch.zeros(4096, dtype=torch.float16).as_strided((1, 2, 64), (3, 64, 1))
        S.sage_rotary(q[:1], None, pos[:1], rotary).backward(strange)
    assert len(taken) == 2 * (4 + 2 + 2) and not any(taken), taken


def test_sizes_whose_products_pass_64_bits():
    for width in (1 << 56, (1 << 55) + 1, 1 << 60, (1 << 63) - 1):
        _refused(_read(width=width, page=256), UNSUPPORTED, "2^30")
        _refused(_attend(width=width, page=256), UNSUPPORTED, "2^30")
    _refused(_read(width=(1 << 26) + 1, page=16), UNSUPPORTED, "2^30")
    size = _native.load().sage_cache_attention_workspace_bytes
    assert size(1, 1 << 40, 1, 1 << 40) == size(1, 2, 1, (1 << 63) - 1) == size(1, 8, 2, (1 << 26) + 1) == 0 and size(1, 8, 2, 1 << 26) > 0
