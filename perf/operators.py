"""The operators around a quantised K/V cache whose speed this package answers for.

Each case is one call as a serving program makes it: inputs already on the GPU, output left there.

  rotary   queries and keys turned to their positions (half or interleaved pairs, part of the head, frequencies
           scaled for long contexts), forward or the transposed map that a gradient takes
  write    new keys and values quantised into the pages of a cache
  read     sequences of the cache read back as packed 16-bit keys and values
  attend   new tokens against the cached keys: one token per sequence, a chain of them, or a tree of drafted ones

Sizes are those of the package's tests and benchmark (288 .. 47520 tokens, 8 .. 48 K/V heads, head_dim 64 .. 128).
Keys carry a bias per channel, which the cache may take off (its shift), and positions reach far beyond the
length that the frequencies were made for.  With `own` false the operators run in their plain form: elementary
torch operations in 32 bits (angles in 64), rounded once at the end.
"""
import math
import os
import random
import sys

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
_E4M3 = torch.float8_e4m3fn
_BASE = dict(kind="attend", b=1, hq=32, hkv=8, n=0, t=1, d=128, page=64, dtype="fp16", int8=True, shift=False,
             mask="chain", ragged=False, lse=False, rot=128, interleaved=False, scaling="none", backward=False)
#: what the largest listed calls move and multiply; nothing drawn goes beyond it
_MOST_BYTES = 4 * 47520 * 48 * 264
_MOST_FLOPS = 4 * 128 * 32 * 8 * 64 * 16384


def _case(name, **kw):
    return dict(_BASE, name=name, **kw)


def listed():
    return [
        # One step of sixteen sequences: their single new tokens, far positions, scaled frequencies. Latency counts.
        _case("rotary_step_16", kind="rotary", b=16, n=1, dtype="bf16", scaling="parts"),
        # A prompt with all heads of the benchmark, half of each head turned, pairs next to each other.
        _case("rotary_prompt_8771_half", kind="rotary", n=8771, hq=48, hkv=48, rot=64, interleaved=True),
        # The gradient of a rotation over a batch of four, grouped heads, bf16.
        _case("rotary_gradient_4x4096", kind="rotary", b=4, n=4096, dtype="bf16", scaling="linear", backward=True),
        # The same step's keys and values into the cache (e4m3 codes, the rule for bf16).
        _case("write_step_16", kind="write", b=16, n=1, dtype="bf16", int8=False),
        # A prompt of ragged length written into scattered pages, channel bias of K taken off.
        _case("write_prompt_8771", kind="write", n=8771, shift=True),
        # Eleven ragged sequences read back for a prefill that continues them.
        _case("read_11_ragged", kind="read", b=11, n=4096, dtype="bf16", int8=False, page=16, ragged=True),
        # A video-length context read back whole, all heads.
        _case("read_27280", kind="read", n=27280, hq=48, hkv=48, page=128, shift=True),
        # One token of one sequence against a long context: nothing to share the cache's reading with.
        _case("decode_1x16384", n=16384),
        # A serving batch of 32 ragged sequences, one of them empty (a padded entry), log-sum-exp wanted.
        _case("decode_32_ragged", b=32, n=8192, dtype="bf16", int8=False, ragged=True, lse=True, page=16),
        # Four video-length contexts, one query head per K/V head: the largest cache.
        _case("decode_4x47520_all_heads", b=4, n=47520, hq=48, hkv=48, page=128, shift=True),
        # A tree of 21 drafted tokens for each of four sequences.
        _case("tree_4x21_8771", b=4, n=8771, t=21, mask="tree", dtype="bf16", ragged=True),
        # A full tree of 64 drafted tokens for each of eight long sequences.
        _case("tree_8x64_16384", b=8, n=16384, t=64, mask="tree", lse=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(["rotary", "write", "read", "attend", "attend", "attend"])
    hkv = rng.choice([4, 8, 12, 16, 24, 40, 48])
    c = dict(_BASE, kind=kind, hkv=hkv, hq=hkv * (rng.choice([1, 2, 4, 8]) if hkv <= 8 else 1),
             d=rng.choice([128, 128, 128, 96, 64]), page=rng.choice([16, 32, 64, 128]), dtype=rng.choice(["fp16", "bf16"]),
             int8=rng.random() < 0.6, shift=rng.random() < 0.4, ragged=rng.random() < 0.5, b=_log_int(rng, 1, 32))
    if kind == "rotary":
        c.update(rot=rng.choice([c["d"], c["d"], c["d"] // 2, 32]), interleaved=rng.random() < 0.5, backward=rng.random() < 0.3,
                 scaling=rng.choice(["none", "linear", "ntk", "parts"]), ragged=False)
        most = 0.25 * _MOST_BYTES / (4 * c["d"] * (c["hq"] + hkv) * c["b"])
        c["n"] = _log_int(rng, 1, min(47520, most))
    elif kind in ("write", "read"):
        c["n"] = _log_int(rng, 1 if kind == "write" else 64, min(47520, 0.25 * _MOST_BYTES / (700 * hkv * c["b"])))
    else:
        c["mask"] = rng.choice(["chain", "tree"])
        c["lse"] = rng.random() < 0.4
        c["t"] = rng.choice([1, 1, _log_int(rng, 2, 96)])
        most = min(0.8 * _MOST_BYTES / (264 * hkv * c["b"]), 0.8 * _MOST_FLOPS / (4 * 128 * c["hq"] * c["t"] * c["b"]))
        c["n"] = _log_int(rng, 128, min(47520, most))
    return c


def _lengths(case):
    """(cached keys, new tokens) of each sequence.  A ragged batch spreads both below their largest and, from four
    sequences on, ends in an empty one: the padding of a serving batch."""
    b, n, t = case["b"], case["n"], case["t"]
    if not case["ragged"]:
        return [n] * b, [t] * b
    rng = random.Random(7919 * n + 31 * b + t)
    keys = [n] + [_log_int(rng, max(1, n // 16), n) for _ in range(b - 1)]
    new = [t] + [rng.randint(1, t) for _ in range(b - 1)]
    if b >= 4 and case["kind"] == "attend":
        keys[-1] = 0
    return keys, new


def _width(d):
    return 64 if d <= 64 else 128


# ---- the formulas, in their plain form ------------------------------------------------------------------------------


def _frequencies(case, dev):
    """(angle per position of each pair in 64 bits, factor on the result), scaled for a context `factor` times as long."""
    rot, factor, trained = case["rot"], 8.0, 4096.0
    i = torch.arange(0, rot, 2, dtype=torch.float64, device=dev) / rot
    base = 10000.0
    if case["scaling"] == "ntk":
        base = base * factor ** (rot / (rot - 2))
    f = base ** -i
    if case["scaling"] == "linear":
        return f / factor, 1.0
    if case["scaling"] == "parts":
        turns = trained * f / (2 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        return f * (keep + (1 - keep) / factor), 0.1 * math.log(factor) + 1.0
    return f, 1.0


def _rotate(x, pos, freq, factor, interleaved, backward):
    """x (tokens, heads, d): the first 2 * len(freq) columns turned, the others as they are."""
    rot = 2 * freq.numel()
    angle = pos.double()[:, None] * freq
    cos, sin = (angle.cos() * factor).float()[:, None], (angle.sin() * factor).float()[:, None]
    if backward:
        sin = -sin
    y = x.float()
    a, b = (y[..., 0:rot:2], y[..., 1:rot:2]) if interleaved else (y[..., :rot // 2], y[..., rot // 2:rot])
    u, w = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((u, w), -1).flatten(-2) if interleaved else torch.cat((u, w), -1)
    return torch.cat((turned, y[..., rot:]), -1).to(x.dtype)


def _quantise(x, int8, width):
    """Rows of x (..., d): codes (..., width) and one scale per row.  Divisions are by tensors, so that they round correctly."""
    most = torch.tensor(127.0 if int8 else 448.0, device=x.device)
    scale = torch.maximum(x.abs().amax(-1) / most, torch.tensor(1e-12, device=x.device))
    y = torch.nn.functional.pad(x / scale[..., None], (0, width - x.shape[-1]))
    codes = y.round().clamp(-128, 127).to(torch.int8) if int8 else y.clamp(-448, 448).to(_E4M3)
    return codes, scale


def _write(s):
    page, off = s["slots"] // s["page"], s["slots"] % s["page"]
    x = s["k"].float()
    if s["shift"] is not None:
        x = x - s["shift"]
    w = s["k_codes"].shape[-1]
    for x, int8, codes, scale in ((x, s["k_codes"].dtype == torch.int8, s["k_codes"], s["k_scale"]),
                                  (s["v"].float(), False, s["v_codes"], s["v_scale"])):
        c, f = _quantise(x, int8, w)
        codes.view(torch.uint8)[page, :, off] = c.view(torch.uint8)
        scale[page, :, off] = f
    return {"k_codes": s["k_codes"], "k_scale": s["k_scale"], "v_codes": s["v_codes"], "v_scale": s["v_scale"]}


def _values(s, name):
    """(b, heads, keys, d) values of the cached rows that the page table names, in 32 bits."""
    codes, scale = s[name + "_codes"], s[name + "_scale"]
    x = codes.view(torch.uint8)[s["table"]].view(codes.dtype).float() * scale[s["table"]][..., None]
    return x.transpose(1, 2).flatten(2, 3)[..., :s["d"]]


def _read(s):
    n = s["table"].shape[1] * s["page"]
    live = torch.arange(n, device=s["keys"].device) < s["keys"][:, None]
    k, v = (_values(s, name).transpose(1, 2)[live] for name in ("k", "v"))
    if s["shift"] is not None:
        k = k + s["shift"]
    return k.to(s["dtype"]), v.to(s["dtype"])


def _attend(s):
    dev, t, hkv = s["q"].device, s["t"], s["k_codes"].shape[1]
    tokens, hq, d = s["q"].shape
    k, v = _values(s, "k"), _values(s, "v")
    b, n = k.shape[0], k.shape[2]
    row = torch.arange(t, device=dev)
    new = s["cu"][1:] - s["cu"][:-1]
    live = row < new[:, None]
    at = (s["cu"][:-1, None] + row).clamp(max=tokens - 1).long()
    q = s["q"].float()[at].view(b, t, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4)
    key = torch.arange(n, device=dev)
    first = s["keys"] - new
    if s["tree"] is None:
        seen = key <= (first[:, None] + row)[..., None]
    else:
        j = (key - first[:, None])[:, None].expand(b, t, n)
        seen = (j < 0) | (s["tree"][at].gather(2, j.clamp(0, t - 1)) & (j < new[:, None, None]))
    seen = (seen & (key < s["keys"][:, None])[:, None])[:, None, None]
    scores = (q.flatten(2, 3) @ k.transpose(2, 3)).view(b, hkv, hq // hkv, t, n) * d ** -0.5
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top.isinf(), 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = (p.flatten(2, 3) @ v).view(b, hkv, hq // hkv, t, d) / torch.where(total > 0, total, 1.0)
    out = torch.empty_like(s["q"])
    out[at[live]] = o.permute(0, 3, 1, 2, 4).flatten(2, 3)[live].to(out.dtype)
    if not s["lse"]:
        return out
    lse = (top + torch.log(total)).squeeze(-1)
    if s["shift"] is not None:
        lse = lse + torch.einsum("bhgtd,hd->bhgt", q, s["shift"]) * d ** -0.5
    res = torch.empty((tokens, hq), dtype=torch.float32, device=dev)
    res[at[live]] = lse.permute(0, 3, 1, 2).flatten(2, 3)[live]
    return out, res


def _package():
    """The package whose operators are measured."""
    at = os.path.join(os.getcwd(), "sageattention-rdna4_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import sageattention
    return sageattention


# ---- what the tools call -------------------------------------------------------------------------------------------


def _randn(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device=gen.device).to(dtype)


def _fill(s, gen, int8, bias):
    """Cached keys and values as an earlier write left them: N(0,1), K with its bias per channel, a few rows much larger."""
    pages, hkv, page, w = s["k_codes"].shape
    for i in range(0, pages, 256):
        shape = (min(256, pages - i), hkv, page, s["d"])
        for name, as_int8, add in (("k", int8, bias), ("v", False, None)):
            x = torch.randn(shape, generator=gen, device=gen.device)
            x *= 1 + 3 * (torch.rand(shape[:3] + (1,), generator=gen, device=gen.device) < 0.02)
            if add is not None:
                x += add[:, None]
            codes, scale = _quantise(x, as_int8, w)
            s[name + "_codes"][i:i + 256].view(torch.uint8).copy_(codes.view(torch.uint8))
            s[name + "_scale"][i:i + 256] = scale


def _tree(gen, new, t):
    """Which drafted tokens each sees: itself and its ancestors; the parent of token j is one of the tokens before it."""
    dev = gen.device
    parent = (torch.rand((len(new), t), generator=gen, device=dev) * torch.arange(t, device=dev)).floor().long()
    sees = torch.eye(t, device=dev).repeat(len(new), 1, 1)
    sees.scatter_(2, parent[..., None], 1.0)
    for _ in range(max(1, math.ceil(math.log2(max(2, t))))):
        sees = ((sees @ sees) > 0).float()
    return torch.cat([sees[i, :m] for i, m in enumerate(new)]) > 0


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(1_000_003 * (seed + 1))
    dt, b, n, d, hq, hkv, page = _DTYPES[case["dtype"]], case["b"], case["n"], case["d"], case["hq"], case["hkv"], case["page"]
    s = {"case": dict(case), "kind": case["kind"], "dtype": dt, "page": page, "d": d, "lse": case["lse"], "t": case["t"]}
    if case["kind"] == "rotary":
        # (positions as they come: steps at unrelated far places, prompts counted up from where they go on)
        start = torch.randint(0, 100_000, (b, 1), generator=gen, device=dev)
        s["pos"] = (start + torch.arange(n, device=dev)).flatten()
        s["q"], s["k"] = _randn(gen, (b * n, hq, d), dt), _randn(gen, (b * n, hkv, d), dt)
        s["freq"], s["factor"] = _frequencies(case, dev)
        if own:
            s["rotary"] = _package().SageRotary(d, rotary_dim=case["rot"], interleaved=case["interleaved"],
                                                scaling=case["scaling"], factor=8.0, original_length=4096, device=dev)
        return s
    keys, new = _lengths(case)
    need = [-(-m // page) for m in keys]
    pages = sum(need) + (need[0] if case["kind"] == "write" and n > 1 else 8)
    w = _width(d)
    s["k_codes"] = torch.zeros((pages, hkv, page, w), dtype=torch.int8 if case["int8"] else _E4M3, device=dev)
    s["v_codes"] = torch.zeros((pages, hkv, page, w), dtype=_E4M3, device=dev)
    s["k_scale"], s["v_scale"] = (torch.zeros((pages, hkv, page), device=dev) for _ in range(2))
    bias = 0.5 * torch.randn((hkv, d), generator=gen, device=dev)
    s["shift"] = bias if case["shift"] else None
    order = torch.randperm(pages, generator=gen, device=dev)
    table = torch.zeros((b, max(need)), dtype=torch.int64, device=dev)
    at = 0
    for i, m in enumerate(need):
        table[i, :m] = order[at:at + m]
        at += m
    s["table"], s["table32"] = table, table.int()
    s["keys"] = torch.tensor(keys, dtype=torch.int32, device=dev)
    if case["kind"] == "write":
        j = torch.arange(max(keys), device=dev)
        live = j < s["keys"][:, None]
        s["slots"] = (table[:, j // page] * page + j % page)[live]
        s["k"] = (torch.randn((sum(keys), hkv, d), generator=gen, device=dev) + bias).to(dt)
        s["v"] = _randn(gen, (sum(keys), hkv, d), dt)
    else:
        _fill(s, gen, case["int8"], None if case["shift"] else bias)
    if case["kind"] == "read":
        s["total"] = sum(keys)
        s["cu"] = torch.tensor([sum(keys[:i]) for i in range(b + 1)], dtype=torch.int32, device=dev)
    if case["kind"] == "attend":
        s["q"] = _randn(gen, (sum(new), hq, d), dt)
        s["cu"] = torch.tensor([sum(new[:i]) for i in range(b + 1)], dtype=torch.int32, device=dev)
        s["tree"] = _tree(gen, new, case["t"]) if case["mask"] == "tree" else None
    if own:
        s["cache"] = _package().SageCache(s["k_codes"], s["k_scale"], s["v_codes"], s["v_scale"], head_dim=d, k_shift=s["shift"])
    return s


def run(s):
    kind, c = s["kind"], s["case"]
    if own:
        sageattention = sys.modules["sageattention"]
        if kind == "rotary":
            return sageattention.sage_rotary(s["q"], s["k"], s["pos"], s["rotary"], backward=c["backward"])
        if kind == "write":
            sageattention.sage_cache_write(s["cache"], s["k"], s["v"], s["slots"])
            return {"k_codes": s["k_codes"], "k_scale": s["k_scale"], "v_codes": s["v_codes"], "v_scale": s["v_scale"]}
        if kind == "read":
            return sageattention.sage_cache_read(s["cache"], s["table32"], s["cu"], s["total"], dtype=s["dtype"])
        return sageattention.sageattn_cached(s["q"], s["cache"], s["table32"], s["keys"], cu_seqlens_q=s["cu"],
                                             max_seqlen_q=s["t"], tree_mask=s["tree"], return_lse=s["lse"])
    if kind == "rotary":
        return tuple(_rotate(x, s["pos"], s["freq"], s["factor"], c["interleaved"], c["backward"]) for x in (s["q"], s["k"]))
    return {"write": _write, "read": _read, "attend": _attend}[kind](s)


def work(case):
    """Each input read once, each output written once; the products of the visible (query, key) pairs."""
    b, n, d, hq, hkv = case["b"], case["n"], case["d"], case["hq"], case["hkv"]
    if case["kind"] == "rotary":
        return {"bytes": b * n * (4 * d * (hq + hkv) + 8), "flops": 3 * b * n * case["rot"] * (hq + hkv)}
    keys, new = _lengths(case)
    rows = sum(keys) * hkv
    coded = 2 * d + 8
    if case["kind"] in ("write", "read"):
        return {"bytes": rows * (4 * d + coded) + 8 * sum(keys), "flops": 4 * rows * d}
    tokens = sum(new)
    pairs = sum(max(0, m - t) * t + min(m, t) * (min(m, t) + 1) // 2 for m, t in zip(keys, new))
    nbytes = rows * coded + 4 * d * hq * tokens + (4 * hq * tokens if case["lse"] else 0)
    return {"bytes": nbytes + (tokens * case["t"] if case["mask"] == "tree" else 0), "flops": 4 * d * hq * pairs}


# ---- the same in 64 bits, written apart from the above -------------------------------------------------------------


def _e4m3_64(y):
    """The nearest value of the format (3 mantissa bits, steps of 2^-9 at least, 448 at most), ties to even."""
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -20))).clamp(min=-6) - 3)
    return (torch.round(y / step) * step).clamp(-448.0, 448.0)


def _exact_rotary(case, s):
    rot, half = case["rot"], case["rot"] // 2
    pairs = [(2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half) for i in range(half)]
    first = torch.tensor([p[0] for p in pairs], device=s["pos"].device)
    second = torch.tensor([p[1] for p in pairs], device=s["pos"].device)
    turn = torch.polar(torch.full((), s["factor"], dtype=torch.float64, device=s["pos"].device),
                       s["pos"].double()[:, None, None] * s["freq"])
    if case["backward"]:
        turn = turn.conj()
    res = []
    for x in (s["q"], s["k"]):
        y = x.double()
        z = torch.complex(y[..., first], y[..., second]) * turn
        y[..., first], y[..., second] = z.real, z.imag
        res.append(y)
    return tuple(res)


def _exact_write(case, s):
    res = {}
    for name, qmax in (("k", 127.0 if case["int8"] else 448.0), ("v", 448.0)):
        x = s[name].double()
        if name == "k" and s["shift"] is not None:
            x = x - s["shift"].double()
        f = torch.clamp(x.abs().amax(-1) / qmax, min=1e-12)
        scale = s[name + "_scale"].double().transpose(1, 2).flatten(0, 1)
        scale[s["slots"]] = f
        pages, hkv = s["k_scale"].shape[:2]
        res[name + "_scale"] = scale.view(pages, s["page"], hkv).transpose(1, 2)
        codes = None
        if qmax == 448.0:
            codes = torch.zeros((pages * s["page"], hkv, s["k_codes"].shape[-1]), dtype=torch.float64, device=x.device)
            codes[s["slots"], :, :case["d"]] = _e4m3_64(x / f[..., None])
            codes = codes.view(pages, s["page"], hkv, -1).transpose(1, 2)
        res[name + "_codes"] = codes
    return res


def _sequence(s, name, i, m):
    """(heads, m, d) values of the first m cached rows of sequence i in 64 bits."""
    ids = s["table"][i, :-(-m // s["page"])]
    x = s[name + "_codes"].view(torch.uint8)[ids].view(s[name + "_codes"].dtype).double() * s[name + "_scale"][ids].double()[..., None]
    return x.permute(1, 0, 2, 3).flatten(1, 2)[:, :m, :s["d"]]


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rotary":
        return _exact_rotary(case, s)
    if case["kind"] == "write":
        return _exact_write(case, s)
    keys, new = _lengths(case)
    if case["kind"] == "read":
        k = torch.cat([_sequence(s, "k", i, m).transpose(0, 1) for i, m in enumerate(keys)])
        v = torch.cat([_sequence(s, "v", i, m).transpose(0, 1) for i, m in enumerate(keys)])
        return (k if s["shift"] is None else k + s["shift"].double()), v
    hq, group, d = case["hq"], case["hq"] // case["hkv"], case["d"]
    out = torch.zeros((sum(new), hq, d), dtype=torch.float64, device="cuda")
    lse = torch.full((sum(new), hq), -math.inf, dtype=torch.float64, device="cuda")
    at = 0
    for i, (m, t) in enumerate(zip(keys, new)):
        if m:
            k, v = _sequence(s, "k", i, m), _sequence(s, "v", i, m)
            hidden = torch.zeros((t, m), dtype=torch.bool, device="cuda")
            own_keys = max(0, m - t)
            drafted = (torch.ones((t, t), device="cuda").tril() > 0) if s["tree"] is None else s["tree"][at:at + t, :t]
            hidden[:, own_keys:] = ~drafted[:, max(0, t - m):]
            for h in range(hq):
                q = s["q"][at:at + t, h].double()
                z = ((q @ k[h // group].T) * d ** -0.5).masked_fill_(hidden, -math.inf)
                e = torch.logsumexp(z, 1)
                fine = torch.where(e.isinf(), 0.0, e)
                out[at:at + t, h] = torch.exp(z - fine[:, None]) @ v[h // group]
                lse[at:at + t, h] = e if s["shift"] is None else e + (q @ s["shift"][h // group].double()) * d ** -0.5
        at += t
    return (out, lse) if case["lse"] else out
