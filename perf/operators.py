"""Performance cases of the attention operators around the quantized GEMMs: rotary positions, the append of
keys and values to a paged cache with the rotation on the way, and attention of new tokens over that cache.

`listed()` holds one case per use, from a single decoded token to a prefill of thousands; `draw()` gives
more of the same ranges. `run` computes a case in plain torch operations in 32 bits where `own` is false,
and through the library's `_async` entry points (torq-tile_amd/tqt_gfx950.py) where it is true.
"""

import ctypes
import importlib.util
import math
import os

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_BOUND = {}
_DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _tqt():
    """The repository's binding and its loaded library."""
    if "lib" not in _BOUND:
        spec = importlib.util.spec_from_file_location(
            "tqt_gfx950", os.path.join(_ROOT, "torq-tile_amd", "tqt_gfx950.py"))
        mod = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(mod)
        _BOUND["mod"], _BOUND["lib"] = mod, mod.load()
    return _BOUND["mod"], _BOUND["lib"]


# ------------------------------------------------------------------------------------------
# Cases
# ------------------------------------------------------------------------------------------

# The heads are those of a model 4096 wide (32 heads of 128 with 8 or 32 for keys and values: the GEMM
# benchmark's k 4096 with n 14336 and 11008), and other usual widths.


def listed():
    return [
        # decode of one sequence: the query heads of one token, where the launch is the cost
        dict(name="rope_decode1", kind="rope", type="f16", tokens=1, heads=32, dim=128, rot=128,
             inter=False, factor=1, max_pos=8192),
        # a prefill chunk of a ragged number of tokens, half of each head rotated, pairs side by
        # side, positions interpolated for a context four times as long
        dict(name="rope_prefill4099", kind="rope", type="bf16", tokens=4099, heads=32, dim=128,
             rot=64, inter=True, factor=4, max_pos=32768),
        # one decode step of 64 sequences: keys and values appended, queries rotated in the same call
        dict(name="append_decode64", kind="append", src="bf16", cache="bf16", tokens=64, heads=32,
             kv_heads=8, dim=128, rot=128, inter=False, page=16, max_pos=8192, slots=8192),
        # a prefill chunk from f32 QKV results (the f32 GEMMs' output) into an f16 cache
        dict(name="append_prefill4096", kind="append", src="f32", cache="f16", tokens=4096,
             heads=32, kv_heads=8, dim=128, rot=128, inter=False, page=64, max_pos=8192,
             slots=8192),
        # a ragged chunk into an int8 cache, as many key heads as query heads
        dict(name="append_int8_1000", kind="append", src="bf16", cache="qsi8dx", tokens=1000,
             heads=32, kv_heads=32, dim=128, rot=128, inter=False, page=32, max_pos=4096,
             slots=1024),
        # one token of one sequence at the end of a long context: the cache's bytes
        dict(name="attn_decode1_long", kind="attn", type="f16", cache="f16", batch=1, q=1,
             kv=131071, ragged=False, heads=32, kv_heads=8, dim=128, page=64, causal=True,
             window=0),
        # a decode batch of 64 sequences of lengths from 2048 to 8192
        dict(name="attn_decode64", kind="attn", type="bf16", cache="bf16", batch=64, q=1, kv=8192,
             ragged=True, heads=32, kv_heads=8, dim=128, page=16, causal=True, window=0),
        # a short decode batch, small contexts: latency
        dict(name="attn_decode4_short", kind="attn", type="f16", cache="f16", batch=4, q=1, kv=500,
             ragged=True, heads=32, kv_heads=8, dim=128, page=16, causal=True, window=0),
        # a decode batch over an int8 cache, as many key heads as query heads
        dict(name="attn_decode32_int8", kind="attn", type="f16", cache="qsi8dx", batch=32, q=1,
             kv=4096, ragged=True, heads=32, kv_heads=32, dim=128, page=32, causal=True, window=0),
        # a chunk of a prompt over what is already in the cache
        dict(name="attn_chunk512", kind="attn", type="f16", cache="f16", batch=1, q=512, kv=8000,
             ragged=False, heads=32, kv_heads=8, dim=128, page=64, causal=True, window=0),
        # a mixed batch: prompts' chunks beside decoded tokens, heads of 64, a sliding window
        dict(name="attn_mixed16", kind="attn", type="bf16", cache="bf16", batch=16, q=512, kv=4096,
             ragged=True, heads=32, kv_heads=4, dim=64, page=16, causal=True, window=1024),
        # a whole prompt from an empty cache: the matrix products
        dict(name="attn_prefill8192", kind="attn", type="bf16", cache="bf16", batch=1, q=8192,
             kv=8192, ragged=False, heads=32, kv_heads=8, dim=128, page=64, causal=True, window=0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


# what a drawn attention case costs at most: multiplications of the padded score matrix in the plain
# form, and values of the cache it gathers (both below the largest listed cases')
_MOST_SCORES = 32 * 8192 * 8192
_MOST_CACHE = 64 * 8192 * 8 * 128


def draw(rng):
    kind = rng.choices(["rope", "append", "attn"], [2, 2, 5])[0]
    dim = rng.choice([64, 80, 96, 128, 128, 128, 192, 256])
    if kind == "rope":
        while True:
            tokens, heads = _log_int(rng, 1, 8192), _log_int(rng, 1, 64)
            if tokens * heads * dim <= 4099 * 32 * 128:
                return dict(kind=kind, type=rng.choice(["f32", "f16", "bf16"]), tokens=tokens,
                            heads=heads, dim=dim, rot=rng.choice([dim, dim, dim // 2, dim - 16]),
                            inter=rng.random() < 0.5, factor=rng.choice([1, 1, 2, 8]),
                            max_pos=rng.choice([2048, 8192, 32768]))
    kv_heads, group = rng.choice([1, 2, 4, 8, 8, 16, 32]), rng.choice([1, 1, 2, 3, 4, 4, 7, 8, 16])
    page = rng.choice([16, 16, 32, 64, 128, 256, 24])
    if kind == "append":
        cache, src = rng.choice([("f16", "f16"), ("bf16", "bf16"), ("f16", "f32"), ("bf16", "f32"),
                                 ("qsi8dx", "f16"), ("qsi8dx", "bf16")])
        while True:
            tokens = _log_int(rng, 1, 4096)
            if tokens * (group + 2) * kv_heads * dim <= 4096 * 48 * 128:
                slots = (tokens + rng.randint(0, 2048)) // page * page + page
                return dict(kind=kind, src=src, cache=cache, tokens=tokens,
                            heads=group * kv_heads, kv_heads=kv_heads, dim=dim,
                            rot=rng.choice([dim, dim, dim // 2]), inter=rng.random() < 0.3,
                            page=page, max_pos=rng.choice([4096, 32768]), slots=slots)
    typ = rng.choice(["f16", "bf16"])
    while True:
        batch = _log_int(rng, 1, 64)
        shape = rng.choice(["decode", "decode", "chunk", "prefill"])
        if shape == "decode":
            q, kv = rng.choice([1, 1, 1, 2, 4]), _log_int(rng, 64, 131072)
        elif shape == "chunk":
            q = _log_int(rng, 8, 1024)
            kv = q + _log_int(rng, 64, 16384)
        else:
            q = kv = _log_int(rng, 16, 8192)
        heads = group * kv_heads
        if (batch * heads * q * kv <= _MOST_SCORES // 2 and
                batch * kv * kv_heads * dim <= _MOST_CACHE // 2):
            causal = shape == "prefill" or rng.random() < 0.8
            return dict(kind="attn", type=typ, cache=rng.choice([typ, typ, "qsi8dx"]), batch=batch,
                        q=q, kv=kv, ragged=batch > 1 and rng.random() < 0.7, heads=heads,
                        kv_heads=kv_heads, dim=dim, page=page, causal=causal,
                        window=_log_int(rng, 128, 4096) if causal and rng.random() < 0.2 else 0)


# ------------------------------------------------------------------------------------------
# Inputs
# ------------------------------------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _table(case):
    """cos | sin of every position, [max_pos, rot] f32, from 64 bits."""
    half = case["rot"] // 2
    i = torch.arange(half, dtype=torch.float64, device="cuda")
    f = 10000.0 ** (-i / half) / case.get("factor", 1)
    a = torch.arange(case["max_pos"], dtype=torch.float64, device="cuda")[:, None] * f
    return torch.cat((torch.cos(a), torch.sin(a)), 1).to(torch.float32)


def _lengths(case):
    """(new tokens, keys) of every sequence: the case's own sizes, or, ragged, keys from a quarter of
    them up and every third sequence with a single new token."""
    got = []
    for b in range(case["batch"]):
        q, kv = case["q"], case["kv"]
        if case["ragged"]:
            x = (0.6180339887 * b) % 1.0
            kv = max(1, int(round(kv * (1 - 0.75 * x))))
            q = min(kv, 1 if b % 3 == 2 else max(1, int(round(q * (1 - 0.9 * x)))))
        got.append((q, kv))
    return got


def _cache_rows(g, shape, cache, typ):
    """Random cache contents: 16-bit values, or int8 with the scale of each token and head."""
    if cache != "qsi8dx":
        return _normal(g, shape, _DTYPE[cache]), None
    pages, page, heads, _ = shape
    x = torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int8)
    s = torch.rand((pages, heads, page), generator=g, device="cuda") * 0.02 + 0.005
    return x, s


def prepare(case, seed):
    g = _generator(seed)
    kind = case["kind"]
    s = dict(case=case)
    if kind == "rope":
        dt = _DTYPE[case["type"]]
        s["x"] = _normal(g, (case["tokens"], case["heads"], case["dim"]), dt)
        s["y"] = torch.empty_like(s["x"])
        s["table"] = _table(case)
        s["pos"] = torch.randint(0, case["max_pos"], (case["tokens"],), generator=g, device="cuda",
                                 dtype=torch.int32)
        return s
    kh, d, page = case["kv_heads"], case["dim"], case["page"]
    if kind == "append":
        src = _DTYPE[case["src"]]
        # one row of the QKV product per token, as the GEMM before leaves it
        n = case["heads"] + 2 * kh
        s["qkv"] = _normal(g, (case["tokens"], n, d), src)
        s["q_out"] = torch.empty((case["tokens"], case["heads"], d), device="cuda",
                                 dtype=_DTYPE[case["cache"]] if case["src"] == "f32" else src)
        s["table"] = _table(case)
        s["pos"] = torch.randint(0, case["max_pos"], (case["tokens"],), generator=g, device="cuda",
                                 dtype=torch.int32)
        pages = case["slots"] // page
        shape = (pages, page, kh, d)
        s["k"], s["sk"] = _cache_rows(g, shape, case["cache"], case["src"])
        s["v"], s["sv"] = _cache_rows(g, shape, case["cache"], case["src"])
        s["slots"] = torch.randperm(pages * page, generator=g, device="cuda")[:case["tokens"]]
        return s
    lengths = _lengths(case)
    dt = _DTYPE[case["type"]]
    s["max_q"], s["max_kv"] = max(q for q, _ in lengths), max(kv for _, kv in lengths)
    starts = [0]
    for q, _ in lengths:
        starts.append(starts[-1] + q)
    s["tokens"] = starts[-1]
    s["q_start"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    s["kv_len"] = torch.tensor([kv for _, kv in lengths], dtype=torch.int32, device="cuda")
    s["q"] = _normal(g, (starts[-1], case["heads"], d), dt, 1.5)
    s["out"] = torch.empty_like(s["q"])
    s["lse"] = torch.empty((starts[-1], case["heads"]), device="cuda")
    per = -(-s["max_kv"] // page)
    pages = case["batch"] * per
    s["table"] = torch.randperm(pages, generator=g, device="cuda").to(torch.int32).reshape(
        case["batch"], per)
    shape = (pages, page, kh, d)
    s["k"], s["sk"] = _cache_rows(g, shape, case["cache"], case["type"])
    s["v"], s["sv"] = _cache_rows(g, shape, case["cache"], case["type"])
    return s


# ------------------------------------------------------------------------------------------
# The plain form: elementary torch operations in 32 bits
# ------------------------------------------------------------------------------------------

def _rotate(x, cos_sin, inter):
    """x [tokens, heads, d] f32 with its first elements rotated in pairs; cos_sin [tokens, rot]."""
    half = cos_sin.shape[1] // 2
    c, s = cos_sin[:, None, :half], cos_sin[:, None, half:]
    if inter:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        r = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        r = torch.cat((a * c - b * s, b * c + a * s), -1)
    return torch.cat((r, x[..., 2 * half:]), -1)


def _plain_rope(s):
    c = s["case"]
    y = _rotate(s["x"].float(), s["table"][s["pos"]], c["inter"])
    return dict(y=y.to(s["x"].dtype))


def _plain_store(cache, scales, rows, slots):
    """rows [tokens, heads, d] f32 into the slots of cache [pages, page, heads, d]."""
    pages, page = cache.shape[:2]
    flat = cache.view(pages * page, *cache.shape[2:])
    if scales is None:
        flat[slots] = rows.to(cache.dtype)
        return
    amax = rows.abs().amax(-1)
    sc = torch.where(amax > 0, amax / 127.0, torch.ones_like(amax))
    flat[slots] = torch.round(rows / sc[..., None]).clamp(-127, 127).to(torch.int8)
    scales[slots // page, :, slots % page] = sc


def _values(cache, scales):
    """The cache's contents as the values they stand for."""
    return cache if scales is None else cache * scales.transpose(1, 2)[..., None]


def _append_outputs(s):
    return dict(q=s["q_out"], k=_values(s["k"], s["sk"]), v=_values(s["v"], s["sv"]))


def _plain_append(s):
    c = s["case"]
    h, kh = c["heads"], c["kv_heads"]
    x = s["qkv"].float()
    qk = _rotate(x[:, :h + kh], s["table"][s["pos"]], c["inter"])
    s["q_out"] = qk[:, :h].to(s["q_out"].dtype)
    _plain_store(s["k"], s["sk"], qk[:, h:], s["slots"])
    _plain_store(s["v"], s["sv"], x[:, h + kh:], s["slots"])
    return _append_outputs(s)


def _plain_attn(s):
    c = s["case"]
    h, kh, d = c["heads"], c["kv_heads"], c["dim"]
    g, nq, nk = h // kh, s["max_q"], s["max_kv"]
    dev = s["q"].device
    start, kv_len = s["q_start"].long(), s["kv_len"].long()
    q_len = start[1:] - start[:-1]
    at = start[:-1, None] + torch.arange(nq, device=dev)
    q = s["q"].float()[at.clamp(max=s["tokens"] - 1)]
    q = q.view(-1, nq, kh, g, d).permute(0, 2, 1, 3, 4).reshape(-1, kh, nq * g, d)
    table = s["table"].long()

    def rows(cache, scales):
        x = _values(cache, scales)[table].float().flatten(1, 2)[:, :nk]
        return x.permute(0, 2, 1, 3).contiguous()

    key = torch.arange(nk, device=dev)
    pos = (kv_len - q_len)[:, None] + torch.arange(nq, device=dev)
    seen = (key < kv_len[:, None, None]).expand(-1, nq, -1)
    if c["causal"]:
        seen = seen & (key <= pos[..., None])
    if c["window"]:
        seen = seen & (key > pos[..., None] - c["window"])
    seen = seen[:, None, :, None, :].expand(-1, 1, -1, g, -1).reshape(-1, 1, nq * g, nk)
    p = torch.matmul(q, rows(s["k"], s["sk"]).transpose(2, 3).contiguous())
    p.mul_(1.0 / math.sqrt(d)).masked_fill_(~seen, -math.inf)
    m = p.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, rows(s["v"], s["sv"])) / torch.where(total > 0, total,
                                                             torch.ones_like(total))
    o = o.view(-1, kh, nq, g, d).permute(0, 2, 1, 3, 4).reshape(-1, nq, h, d)
    lse = (m + torch.log(total)).view(-1, kh, nq, g).permute(0, 2, 1, 3).reshape(-1, nq, h)
    token = torch.arange(s["tokens"], device=dev)
    seq = torch.searchsorted(start[1:], token, right=True)
    i = token - start[seq]
    return dict(out=o[seq, i].to(s["q"].dtype), lse=lse[seq, i])


# ------------------------------------------------------------------------------------------
# The library's calls
# ------------------------------------------------------------------------------------------

def _map(mod, s):
    c = s["case"]
    return mod.RopeMap(table=s["table"].data_ptr(), max_pos=c["max_pos"], rotary_dim=c["rot"],
                       interleaved=int(c["inter"]), inverse=0)


def _paged(mod, s):
    k, c = s["k"], s["case"]
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    return mod.PagedKV(k=ptr(k), v=ptr(s["v"]), scale_k=ptr(s["sk"]), scale_v=ptr(s["sv"]),
                       num_pages=k.shape[0], page_size=c["page"], kv_heads=c["kv_heads"],
                       head_dim=c["dim"], page_stride=k.stride(0), token_stride=k.stride(1),
                       head_stride=k.stride(2))


def _plan(s):
    """The entry point and its arguments, which a program builds once for its buffers."""
    mod, lib = _tqt()
    c = s["case"]
    d = c["dim"]
    if c["kind"] == "rope":
        row = c["heads"] * d
        p = mod.RopeParams(tokens=c["tokens"], heads=c["heads"], head_dim=d, X=s["x"].data_ptr(),
                           x_token_stride=row, x_head_stride=d, Y=s["y"].data_ptr(),
                           y_token_stride=row, y_head_stride=d, positions=s["pos"].data_ptr(),
                           map=_map(mod, s))
        return lib.op("rope_" + c["type"], "run_async"), p, dict(y=s["y"])
    if c["kind"] == "append":
        h, kh, x = c["heads"], c["kv_heads"], s["qkv"]
        row, base = x.stride(0), x.data_ptr()
        step = d * x.element_size()
        p = mod.KVAppendRopeParams(
            tokens=c["tokens"], K=base + h * step, k_token_stride=row, k_head_stride=d,
            V=base + (h + kh) * step, v_token_stride=row, v_head_stride=d, q_heads=h, Q=base,
            q_token_stride=row, q_head_stride=d, Q_out=s["q_out"].data_ptr(),
            qo_token_stride=h * d, qo_head_stride=d, positions=s["pos"].data_ptr(),
            slots=s["slots"].data_ptr(), map=_map(mod, s), kv=_paged(mod, s))
        return lib.op("kv_append_rope_%s_%s" % (c["cache"], c["src"]), "run_async"), p, None
    h = c["heads"]
    p = mod.AttnPagedParams(
        batch=c["batch"], q_tokens=s["tokens"], q_heads=h, max_q_len=s["max_q"],
        max_kv_len=s["max_kv"], Q=s["q"].data_ptr(), q_token_stride=h * d, q_head_stride=d,
        D=s["out"].data_ptr(), d_token_stride=h * d, d_head_stride=d, lse=s["lse"].data_ptr(),
        q_start=s["q_start"].data_ptr(), kv_len=s["kv_len"].data_ptr(),
        block_table=s["table"].data_ptr(), ld_table=s["table"].stride(0),
        scale=1.0 / math.sqrt(d), causal=int(c["causal"]), window=c["window"], kv=_paged(mod, s))
    size = lib.op("attn_paged", "get_workspace_size")(ctypes.byref(p))
    s["workspace"] = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
    p.workspace, p.workspace_size = s["workspace"].data_ptr(), size
    return (lib.op("attn_paged_%s_%s" % (c["type"], c["cache"]), "run_async"), p,
            dict(out=s["out"], lse=s["lse"]))


def run(state):
    if not own:
        return {"rope": _plain_rope, "append": _plain_append,
                "attn": _plain_attn}[state["case"]["kind"]](state)
    if "plan" not in state:
        state["plan"] = _plan(state)
    f, p, out = state["plan"]
    f(ctypes.byref(p), torch.cuda.current_stream().cuda_stream)
    return out if out is not None else _append_outputs(state)


# ------------------------------------------------------------------------------------------
# What a pass cannot do without
# ------------------------------------------------------------------------------------------

_SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def _seen(case, q, kv):
    """(pairs of a query and a key it sees, keys that any query sees) of one sequence."""
    first = kv - q
    if not case["causal"]:
        return q * kv, kv
    w = case["window"] or kv
    pairs = 0
    short = max(0, min(q, w - first))  # queries whose window reaches the start
    pairs += short * first + short * (short + 1) // 2
    pairs += (q - short) * w
    return pairs, kv - max(0, first + 1 - w)


def work(case):
    d = case["dim"]
    if case["kind"] == "rope":
        n = case["tokens"] * case["heads"] * d
        return dict(bytes=2 * n * _SIZE[case["type"]] + case["tokens"] * 4 * (case["rot"] + 1),
                    flops=3 * case["tokens"] * case["heads"] * case["rot"])
    h, kh = case["heads"], case["kv_heads"]
    if case["kind"] == "append":
        t = case["tokens"]
        row = d + 4 if case["cache"] == "qsi8dx" else 2 * d
        b = t * (h + 2 * kh) * d * _SIZE[case["src"]] + t * h * d * 2 + 2 * t * kh * row
        if case["cache"] == "qsi8dx":  # returned as the values it stands for
            b += 2 * case["slots"] * kh * (row + 4 * d)
        return dict(bytes=b + t * (4 * case["rot"] + 12), flops=3 * t * (h + kh) * case["rot"])
    row = d + 4 if case["cache"] == "qsi8dx" else 2 * d
    lengths = [(q, kv) + _seen(case, q, kv) for q, kv in _lengths(case)]
    tokens = sum(x[0] for x in lengths)
    return dict(bytes=tokens * h * (4 * d + 4) + 2 * kh * row * sum(x[3] for x in lengths),
                flops=4 * d * h * sum(x[2] for x in lengths))


# ------------------------------------------------------------------------------------------
# The same results in 64 bits
# ------------------------------------------------------------------------------------------

def _exact_rotation(x, case, s):
    """x [tokens, heads, d] f64: every pair as a complex number, times cos + i sin."""
    r = case["rot"]
    t = s["table"].double()[s["pos"].long()]
    w = torch.complex(t[:, :r // 2], t[:, r // 2:])[:, None]
    head = x[..., :r].reshape(*x.shape[:2], *((r // 2, 2) if case["inter"] else (2, r // 2)))
    if not case["inter"]:
        head = head.transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(head.contiguous()) * w)
    if not case["inter"]:
        z = z.transpose(-1, -2)
    out = x.clone()
    out[..., :r] = z.reshape(*x.shape[:2], r)
    return out


def _exact_append(case, s):
    h, kh, page = case["heads"], case["kv_heads"], case["page"]
    x = s["qkv"].double()
    x[:, :h + kh] = _exact_rotation(x[:, :h + kh].clone(), case, s)
    out = dict(q=x[:, :h])
    for name, scale, rows in (("k", "sk", x[:, h:h + kh]), ("v", "sv", x[:, h + kh:])):
        old = s[name].double()
        if s[scale] is not None:
            old = old * s[scale].double().permute(0, 2, 1).unsqueeze(-1)
            step = rows.abs().max(-1, keepdim=True).values / 127
            rows = torch.where(step > 0, torch.round(rows / step) * step, torch.zeros_like(rows))
        old[s["slots"] // page, s["slots"] % page] = rows
        out[name] = old
    return out


def _exact_attn(case, s):
    h, kh, d = case["heads"], case["kv_heads"], case["dim"]
    out = torch.zeros((s["tokens"], h, d), dtype=torch.float64, device="cuda")
    lse = torch.zeros((s["tokens"], h), dtype=torch.float64, device="cuda")
    first = 0
    for b, (nq, nk) in enumerate(_lengths(case)):
        pages = s["table"][b, :-(-nk // case["page"])].long()
        past = (nk - nq + torch.arange(nq, device="cuda"))[:, None]
        key = torch.arange(nk, device="cuda")[None]
        hidden = torch.zeros((nq, nk), dtype=torch.bool, device="cuda")
        if case["causal"]:
            hidden |= key > past
        if case["window"]:
            hidden |= key <= past - case["window"]
        for j in range(kh):
            kv = []
            for name, scale in (("k", "sk"), ("v", "sv")):
                rows = s[name][pages, :, j].double()
                if s[scale] is not None:
                    rows = rows * s[scale][pages, j].double()[..., None]
                kv.append(rows.reshape(-1, d)[:nk])
            for i in range(j * (h // kh), (j + 1) * (h // kh)):
                q = s["q"][first:first + nq, i].double()
                a = (q @ kv[0].T) / math.sqrt(d)
                a[hidden] = -math.inf
                out[first:first + nq, i] = torch.softmax(a, -1) @ kv[1]
                lse[first:first + nq, i] = torch.logsumexp(a, -1)
        first += nq
    return dict(out=out, lse=lse)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rope":
        return dict(y=_exact_rotation(s["x"].double(), case, s))
    return (_exact_append if case["kind"] == "append" else _exact_attn)(case, s)
