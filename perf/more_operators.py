"""Performance cases of a serving step with drafted tokens over the paged cache: the step's bookkeeping (pages,
block tables, slots, positions, masks of drafted trees), the norm of query and key heads with their rotation
(alone, its gradient, and on the way into the cache), attention of a tree of drafted tokens, and the cache's
rows of the tokens that were accepted.

`listed()` holds one case per use; `draw()` gives more of the same ranges. `run` computes a case in plain
torch operations in 32 bits where `own` is false, and through the library's `_async` entry points
(torq-tile_amd/tqt_gfx950.py) where it is true.
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
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}


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

# The heads are those of a model 4096 wide (32 heads of 128 with 8 or 32 for keys and values), as in the cases
# of the paged cache without trees.


def listed():
    return [
        # the query heads of one decoded token, normalised and rotated: the launch is the cost
        dict(name="norm_decode1", kind="norm", type="f16", tokens=1, heads=32, dim=128, rot=128, inter=False,
             shift=0.0, grad=False, max_pos=8192),
        # fine-tuning a few heads in f32 over a short batch: forward, gradients of rows and weight
        dict(name="norm_train200_f32", kind="norm", type="f32", tokens=200, heads=8, dim=80, rot=80, inter=True,
             shift=1.0, grad=True, max_pos=2048),
        # a training step's ragged number of tokens, half of each head rotated: forward and gradients
        dict(name="norm_train4099", kind="norm", type="bf16", tokens=4099, heads=32, dim=128, rot=64, inter=False,
             shift=0.0, grad=True, max_pos=8192),
        # one decode step of 64 sequences: heads of Q and K normalised and rotated, K and V appended
        dict(name="append_norm_decode64", kind="append", src="bf16", cache="bf16", tokens=64, heads=32, kv_heads=8,
             dim=128, rot=128, inter=False, shift=0.0, page=16, max_pos=8192, slots=8192),
        # a prefill chunk from the f32 results of the QKV product into an f16 cache
        dict(name="append_norm_prefill4096", kind="append", src="f32", cache="f16", tokens=4096, heads=32,
             kv_heads=8, dim=128, rot=128, inter=False, shift=0.0, page=64, max_pos=8192, slots=8192),
        # pages, slots and tree masks of 64 sequences with trees of 8 to 26 drafted tokens, a few of them ended
        dict(name="plan_tree64", kind="plan", batch=64, new=26, kv=4096, page=16, tree=True, ended=5),
        # a mixed step of 256 sequences: prompts' chunks beside decoded tokens
        dict(name="plan_mixed256", kind="plan", batch=256, new=300, kv=8192, page=16, tree=False, ended=9),
        # accepted rows of one layer's cache of one sequence: latency
        dict(name="keep1", kind="keep", cache="f16", batch=1, nodes=7, kv=500, accepted=3, layers=1, kv_heads=8,
             dim=128, page=16),
        # accepted rows of 64 sequences in eight layers at once
        dict(name="keep64_layers8", kind="keep", cache="bf16", batch=64, nodes=26, kv=200, accepted=5, layers=8,
             kv_heads=8, dim=128, page=16),
        # a small tree over a short context: latency
        dict(name="tree1_short", kind="tree", type="f16", cache="f16", batch=1, nodes=7, kv=1000, ragged=False,
             heads=32, kv_heads=8, dim=128, page=16, window=0),
        # 64 sequences of 2048 to 8192 keys with trees of up to 8 tokens: the cache's bytes
        dict(name="tree64", kind="tree", type="bf16", cache="bf16", batch=64, nodes=8, kv=8192, ragged=True,
             heads=32, kv_heads=8, dim=128, page=16, window=0),
        # large trees over long contexts in an int8 cache: bytes and matrix products together
        dict(name="tree16_int8", kind="tree", type="f16", cache="qsi8dx", batch=16, nodes=63, kv=16384,
             ragged=True, heads=32, kv_heads=8, dim=128, page=64, window=0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


# what a drawn attention case costs at most: scores of the plain form, and values of the cache it gathers
_MOST_SCORES = 16 * 32 * 63 * 16384
_MOST_CACHE = 64 * 8192 * 8 * 128


def draw(rng):
    kind = rng.choices(["norm", "append", "plan", "keep", "tree"], [2, 2, 2, 1, 5])[0]
    dim = rng.choice([64, 80, 96, 128, 128, 128, 192, 256])
    rot = rng.choice([dim, dim, dim, dim // 2])
    if kind == "norm":
        while True:
            tokens, heads = _log_int(rng, 1, 8192), _log_int(rng, 1, 64)
            if tokens * heads * dim <= 4099 * 32 * 128:
                return dict(kind=kind, type=rng.choice(["f32", "f16", "bf16"]), tokens=tokens, heads=heads, dim=dim,
                            rot=rot, inter=rng.random() < 0.5, shift=rng.choice([0.0, 0.0, 1.0]),
                            grad=rng.random() < 0.5, max_pos=rng.choice([2048, 8192, 32768]))
    if kind == "plan":
        tree = rng.random() < 0.5
        while True:
            batch, new = _log_int(rng, 1, 1024), _log_int(rng, 1, 128 if tree else 4096)
            kv, page = _log_int(rng, 16, 32768), rng.choice([16, 16, 32, 64, 24])
            if batch * new <= 32768 and batch * (kv + new) // page <= 1 << 20:
                return dict(kind=kind, batch=batch, new=new, kv=kv, page=page, tree=tree,
                            ended=rng.randint(0, batch // 2))
    kv_heads, group = rng.choice([1, 2, 4, 8, 8, 16, 32]), rng.choice([1, 1, 2, 3, 4, 4, 7, 8, 16])
    page = rng.choice([16, 16, 32, 64, 128, 256, 24])
    if kind == "append":
        cache, src = rng.choice([("f16", "f16"), ("bf16", "bf16"), ("f16", "f32"), ("bf16", "f32"),
                                 ("qsi8dx", "f16"), ("qsi8dx", "bf16")])
        while True:
            tokens = _log_int(rng, 1, 4096)
            if tokens * (group + 2) * kv_heads * dim <= 4096 * 48 * 128:
                slots = (tokens + rng.randint(0, 2048)) // page * page + page
                return dict(kind=kind, src=src, cache=cache, tokens=tokens, heads=group * kv_heads,
                            kv_heads=kv_heads, dim=dim, rot=rot, inter=rng.random() < 0.3,
                            shift=rng.choice([0.0, 0.0, 1.0]), page=page, max_pos=rng.choice([4096, 32768]),
                            slots=slots)
    if kind == "keep":
        while True:
            batch, nodes, layers = _log_int(rng, 1, 64), _log_int(rng, 2, 64), _log_int(rng, 1, 16)
            kv = nodes + _log_int(rng, 16, 1024)
            if batch * layers * (kv + page) * kv_heads * dim <= 64 * 8 * 216 * 8 * 128:
                return dict(kind=kind, cache=rng.choice(["f16", "bf16", "qsi8dx"]), batch=batch, nodes=nodes, kv=kv,
                            accepted=rng.randint(1, min(8, nodes)), layers=layers, kv_heads=kv_heads, dim=dim,
                            page=page)
    typ = rng.choice(["f16", "bf16"])
    while True:
        batch, nodes = _log_int(rng, 1, 64), _log_int(rng, 1, 128)
        kv = nodes + _log_int(rng, 32, 131072)
        if (batch * group * kv_heads * nodes * kv <= _MOST_SCORES // 2 and
                batch * kv * kv_heads * dim <= _MOST_CACHE // 2):
            return dict(kind=kind, type=typ, cache=rng.choice([typ, typ, "qsi8dx"]), batch=batch, nodes=nodes,
                        kv=kv, ragged=batch > 1 and rng.random() < 0.7, heads=group * kv_heads,
                        kv_heads=kv_heads, dim=dim, page=page,
                        window=_log_int(rng, 128, 4096) if rng.random() < 0.2 else 0)


# ------------------------------------------------------------------------------------------
# Inputs
# ------------------------------------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _table(case):
    """cos | sin of every position, [max_pos, rot] f32, from 64 bits."""
    half = case["rot"] // 2
    i = torch.arange(half, dtype=torch.float64, device="cuda")
    a = torch.arange(case["max_pos"], dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (-i / half)
    return torch.cat((torch.cos(a), torch.sin(a)), 1).to(torch.float32)


def _weight(g, case):
    """A trained norm's weight: around 1, shift and all."""
    return 1.0 - case["shift"] + 0.1 * torch.randn(case["dim"], generator=g, device="cuda")


def _cache_rows(g, shape, cache):
    """Random cache contents: 16-bit values, or int8 with the scale of each token and head. shape: [..., pages,
    page, heads, d]."""
    if cache != "qsi8dx":
        return _normal(g, shape, _DTYPE[cache]), None
    x = torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int8)
    s = torch.rand(shape[:-3] + (shape[-2], shape[-3]), generator=g, device="cuda") * 0.02 + 0.005
    return x, s


def _spread(b):
    return (0.6180339887 * b) % 1.0


def _lengths(case):
    """(drafted tokens, keys with them) of every sequence: the case's own sizes, or, ragged, from a quarter of the
    keys up, and from a third of the nodes."""
    got = []
    for b in range(case["batch"]):
        n, kv = case["nodes"], case["kv"]
        if case.get("ragged"):
            kv = max(1, int(round(kv * (1 - 0.75 * _spread(b)))))
            n = min(kv, max(1, int(round(n * (1 - 0.66 * _spread(3 * b + 1))))))
        got.append((n, kv))
    return got


def _starts(lengths):
    total, got = 0, [0]
    for n in lengths:
        total += n
        got.append(total)
    return got


def _parents(g, starts):
    """Trees in the order of drafting: the first token of a sequence follows its context, each other one some
    token before it."""
    start = _ints(starts, torch.int64)
    row = torch.arange(starts[-1], device="cuda")
    i = row - start[torch.searchsorted(start[1:].contiguous(), row, right=True)]
    u = torch.rand(starts[-1], generator=g, device="cuda")
    return torch.where(i > 0, (u * i).long().clamp(max=starts[-1]), -1).to(torch.int32)


def _ancestors(parent, start, most):
    """[rows, most] 32-bit 0 / 1: whether a row's token is token t of its sequence or descends from it, and the
    rows' number among them. start [batch + 1] 64-bit."""
    rows = parent.shape[0]
    row = torch.arange(rows, device="cuda")
    seq = torch.searchsorted(start[1:].contiguous(), row, right=True).clamp(max=start.shape[0] - 2)
    i = row - start[seq]
    batch = start.shape[0] - 1
    link = torch.zeros((batch, most, most), device="cuda")
    link[seq, i, parent.long().clamp(min=0)] = (parent >= 0).float()
    reach = link + torch.eye(most, device="cuda")
    for _ in range(max(1, (most - 1).bit_length())):  # paths of twice the length
        reach = (torch.matmul(reach, reach) > 0).float()
    return reach[seq, i], i


def _pack(bits):
    """[rows, n] 0 / 1 as 32-bit words, lowest bit first."""
    rows, n = bits.shape
    words = -(-n // 32)
    x = torch.zeros((rows, words * 32), dtype=torch.int64, device="cuda")
    x[:, :n] = bits.long()
    x = (x.view(rows, words, 32) << torch.arange(32, device="cuda")).sum(-1)
    return torch.where(x >= 1 << 31, x - (1 << 32), x).to(torch.int32)


def _prepare_plan(case, g, s):
    """A step's lengths: a third of the sequences decode one token (or draft a small tree), the others take up to
    `new`; some have just ended. Pages are those that the held tokens need, now and then one more."""
    batch, page = case["batch"], case["page"]
    new, kv, held = [], [], []
    for b in range(batch):
        x = _spread(b)
        n = max(1, int(round(case["new"] * (1 - 0.7 * x))))
        new.append(-1 if b % (batch // max(1, case["ended"]) + 1) == 1 and case["ended"] else
                   n if case["tree"] or b % 3 else 1)
        kv.append(max(1, int(round(case["kv"] * (1 - 0.9 * _spread(2 * b + 1))))))
        held.append(-(-kv[-1] // page) + (b % 5 == 0))
    most = max(max(new), 1)
    s["most"], s["tokens"] = most, sum(max(n, 0) for n in new)
    ld = -(-(case["kv"] + case["new"]) // page) + 1
    used = sum(held)
    need = sum(max(0, -(-(k + max(n, 0)) // page) - h) for k, n, h in zip(kv, new, held))
    pages = used + need + 64
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    s["new_len"], s["kv_len"], s["held"] = _ints(new), _ints(kv), _ints(held)
    # the batch's pages in their rows, the others on the stack of free ones
    col = torch.arange(ld, device="cuda")
    at = (torch.cumsum(s["held"], 0) - s["held"])[:, None] + col
    s["table"] = torch.where(col < s["held"][:, None], order[at.clamp(max=used - 1)],
                             torch.full_like(at, -1).to(torch.int32))
    s["free"] = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
    s["free"][:pages - used] = order[used:]
    s["free_count"] = _ints([pages - used])
    s["pages"], s["words"] = pages, -(-most // 32)
    s["parent"] = None
    if case["tree"]:
        s["parent"] = _parents(g, _starts([max(n, 0) for n in new]))
    out = {"kv_len_out": batch, "held_out": batch, "free_count_out": 1, "refused": 1, "q_start": batch + 1,
           "positions": s["tokens"]}
    s["out"] = {k: torch.empty(n, dtype=torch.int32, device="cuda") for k, n in out.items()}
    s["out"]["slots"] = torch.empty(s["tokens"], dtype=torch.int64, device="cuda")
    if case["tree"]:
        s["out"]["mask"] = torch.empty((s["tokens"], s["words"]), dtype=torch.int32, device="cuda")
    return s


def prepare(case, seed):
    g = _generator(seed)
    kind = case["kind"]
    s = dict(case=case)
    if kind == "plan":
        return _prepare_plan(case, g, s)
    d = case["dim"]
    if kind == "norm":
        shape = (case["tokens"], case["heads"], d)
        s["x"] = _normal(g, shape, _DTYPE[case["type"]], 2.0)
        s["dy"] = _normal(g, shape, _DTYPE[case["type"]], 0.5)
        s["y"], s["dx"] = torch.empty_like(s["x"]), torch.empty_like(s["x"])
        s["w"], s["table"] = _weight(g, case), _table(case)
        s["dw"] = torch.empty(d, device="cuda")
        s["pos"] = torch.randint(0, case["max_pos"], shape[:1], generator=g, device="cuda", dtype=torch.int32)
        return s
    kh, page = case["kv_heads"], case["page"]
    if kind == "append":
        # one row of the QKV product per token, as the GEMM before leaves it
        n = case["heads"] + 2 * kh
        s["qkv"] = _normal(g, (case["tokens"], n, d), _DTYPE[case["src"]], 2.0)
        s["q_out"] = torch.empty((case["tokens"], case["heads"], d), device="cuda",
                                 dtype=_DTYPE[case["cache"] if case["src"] == "f32" else case["src"]])
        s["wq"], s["wk"], s["table"] = _weight(g, case), _weight(g, case), _table(case)
        s["pos"] = torch.randint(0, case["max_pos"], (case["tokens"],), generator=g, device="cuda",
                                 dtype=torch.int32)
        pages = case["slots"] // page
        for k, sk in (("k", "sk"), ("v", "sv")):
            s[k], s[sk] = _cache_rows(g, (pages, page, kh, d), case["cache"])
        s["slots"] = torch.randperm(pages * page, generator=g, device="cuda")[:case["tokens"]]
        return s
    lengths = _lengths(case)
    starts = _starts([n for n, _ in lengths])
    s["max_q"], s["max_kv"] = max(n for n, _ in lengths), max(kv for _, kv in lengths)
    s["tokens"], s["q_start"] = starts[-1], _ints(starts)
    s["kv_len"] = _ints([kv for _, kv in lengths])
    per = -(-s["max_kv"] // page)
    pages = case["batch"] * per
    s["table"] = torch.randperm(pages, generator=g, device="cuda").to(torch.int32).reshape(case["batch"], per)
    lead = (case["layers"],) if kind == "keep" else ()
    for k, sk in (("k", "sk"), ("v", "sv")):
        s[k], s[sk] = _cache_rows(g, lead + (pages, page, kh, d), case["cache"])
    if kind == "keep":
        # an accepted path: the first token, then ever later ones, past the rows that the path will fill (so that
        # a second pass over the same state moves the same rows)
        nodes, most = case["nodes"], case["accepted"]
        n = torch.randint(1, most + 1, (case["batch"],), generator=g, device="cuda", dtype=torch.int32)
        rest = max(nodes - most, 0)
        u = torch.rand((case["batch"], max(rest, 1)), generator=g, device="cuda")
        late = most + torch.sort(torch.argsort(u, 1)[:, :most - 1], 1).values
        path = torch.cat((torch.zeros_like(late[:, :1]) if late.shape[1] else
                          torch.zeros((case["batch"], 1), dtype=torch.int64, device="cuda"), late), 1)
        s["keep"] = path.clamp(max=nodes - 1).to(torch.int32).contiguous()
        s["keep_len"] = n.clamp(max=min(s["keep"].shape[1], 1 + rest)).to(torch.int32)
        s["kv_len_out"] = torch.empty(case["batch"], dtype=torch.int32, device="cuda")
        return s
    dt = _DTYPE[case["type"]]
    s["q"] = _normal(g, (starts[-1], case["heads"], d), dt, 1.5)
    s["out"] = torch.empty_like(s["q"])
    s["lse"] = torch.empty((starts[-1], case["heads"]), device="cuda")
    s["mask"] = _pack(_ancestors(_parents(g, starts), s["q_start"].long(), s["max_q"])[0])
    return s


# ------------------------------------------------------------------------------------------
# The plain form: elementary torch operations in 32 bits
# ------------------------------------------------------------------------------------------

_EPS = 1e-6


def _turn(x, cos_sin, inter, sign=1.0):
    """x [tokens, heads, d] f32 with its first elements turned in pairs; cos_sin [tokens, rot]."""
    half = cos_sin.shape[1] // 2
    c, s = cos_sin[:, None, :half], cos_sin[:, None, half:] * sign
    if inter:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        r = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        r = torch.cat((a * c - b * s, b * c + a * s), -1)
    return torch.cat((r, x[..., 2 * half:]), -1)


def _normed(x, factor):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS) * factor


def _plain_norm(s):
    c = s["case"]
    x, factor, t = s["x"].float(), s["w"] + c["shift"], s["table"][s["pos"]]
    out = dict(y=_turn(_normed(x, factor), t, c["inter"]).to(s["x"].dtype))
    if c["grad"]:
        u = _turn(s["dy"].float(), t, c["inter"], -1.0)
        r = torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS)
        n = x * r
        fu = u * factor
        out["dx"] = ((fu - n * (fu * n).mean(-1, keepdim=True)) * r).to(s["x"].dtype)
        out["dw"] = (u * n).double().sum((0, 1)).float()
    return out


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


def _values(cache, scales, dtype=None):
    """The cache's contents as the values they stand for."""
    if scales is None:
        return cache
    x = cache * scales.transpose(-1, -2)[..., None]
    return x if dtype is None else x.to(dtype)


def _append_outputs(s):
    dt = s["qkv"].dtype
    return dict(q=s["q_out"], k=_values(s["k"], s["sk"], dt), v=_values(s["v"], s["sv"], dt))


def _plain_append(s):
    c = s["case"]
    h, kh = c["heads"], c["kv_heads"]
    x, t = s["qkv"].float(), s["table"][s["pos"]]
    s["q_out"] = _turn(_normed(x[:, :h], s["wq"] + c["shift"]), t, c["inter"]).to(s["q_out"].dtype)
    _plain_store(s["k"], s["sk"], _turn(_normed(x[:, h:h + kh], s["wk"] + c["shift"]), t, c["inter"]), s["slots"])
    _plain_store(s["v"], s["sv"], x[:, h + kh:], s["slots"])
    return _append_outputs(s)


def _plain_plan(s):
    c = s["case"]
    page, ld, tokens = c["page"], s["table"].shape[1], s["tokens"]
    new, kv, held = s["new_len"].long(), s["kv_len"].long(), s["held"].long()
    ended, n = new < 0, new.clamp(min=0)
    rows = torch.cumsum(n, 0)
    # pages of ended sequences go on the stack in order, then new ones come from its top
    col = torch.arange(ld, device="cuda")
    back = ended[:, None] & (col < held[:, None]) & (s["table"] >= 0) & (s["table"] < s["pages"])
    count = s["free_count"].long()
    last = s["free"].shape[0]
    to = torch.where(back.flatten(), count + torch.cumsum(back.flatten().long(), 0) - 1, last).clamp(max=last)
    stack = torch.cat((s["free"], s["free"][:1])).index_put((to,), s["table"].flatten())[:-1]
    top = (count + back.sum()).clamp(max=last)
    need = ((kv + n + page - 1) // page - held).clamp(min=0)
    fits = ~ended & (rows <= tokens) & (held + need <= ld)
    need = torch.where(fits, need, 0)
    upto = torch.cumsum(need, 0)
    served = fits & ((need == 0) | (upto <= top))
    take = torch.where(served, need, 0)
    fresh = served[:, None] & (col >= held[:, None]) & (col < (held + take)[:, None])
    at = top - 1 - ((upto - need - held)[:, None] + col)
    table = torch.where(fresh, stack[at.clamp(0, last - 1)], s["table"])
    row = torch.arange(tokens, device="cuda")
    seq = torch.searchsorted(rows, row, right=True).clamp(max=rows.shape[0] - 1)
    i = row - (rows - n)[seq]
    here = kv[seq] + i
    p = table[seq, (here // page).clamp(max=ld - 1)].long()
    slots = torch.where(served[seq] & (p >= 0) & (p < s["pages"]), p * page + here % page, -1)
    out = dict(kv_len_out=torch.where(ended, 0, torch.where(served, kv + n, kv)),
               held_out=torch.where(ended, 0, held + take), free_count_out=top - take.sum(),
               refused=(~ended & ~served).sum().reshape(1), q_start=torch.cat((rows[:1] * 0, rows)).clamp(max=tokens))
    if s["parent"] is not None:
        bits, _ = _ancestors(s["parent"], out["q_start"], s["most"])
        out["mask"] = _pack(bits)
        here = kv[seq] + bits.sum(-1).long() - 1
    out["positions"] = here
    out = {k: v.to(torch.int32) for k, v in out.items()}
    return dict(out, slots=slots, table=table, free=stack)


def _plain_keep(s):
    c = s["case"]
    page = c["page"]
    n_q = (s["q_start"][1:] - s["q_start"][:-1]).long()
    base = s["kv_len"].long() - n_q
    j = torch.arange(s["keep"].shape[1], device="cuda")
    kept = j < s["keep_len"][:, None]
    src = base[:, None] + torch.where(kept, s["keep"].long(), j.clamp(max=c["nodes"] - 1))
    dst = base[:, None] + torch.where(kept, j, j.clamp(max=c["nodes"] - 1))
    table = s["table"].long()
    b = torch.arange(c["batch"], device="cuda")[:, None]
    sp, so, tp, to = table[b, src // page], src % page, table[b, dst // page], dst % page
    for name in ("k", "v"):
        s[name][:, tp, to] = s[name][:, sp, so]
        if s["s" + name] is not None:
            s["s" + name][:, tp, :, to] = s["s" + name][:, sp, :, so]
    return _keep_outputs(s, (base + s["keep_len"]).to(torch.int32))


def _keep_outputs(s, kv_len_out):
    return dict(k=_values(s["k"], s["sk"], torch.float16), v=_values(s["v"], s["sv"], torch.float16),
                kv_len=kv_len_out)


def _plain_tree(s):
    c = s["case"]
    h, kh, d = c["heads"], c["kv_heads"], c["dim"]
    g, nq, nk = h // kh, s["max_q"], s["max_kv"]
    start, kv_len = s["q_start"].long(), s["kv_len"].long()
    q_len = start[1:] - start[:-1]
    at = (start[:-1, None] + torch.arange(nq, device="cuda")).clamp(max=s["tokens"] - 1)
    q = s["q"].float()[at]
    q = q.view(-1, nq, kh, g, d).permute(0, 2, 1, 3, 4).reshape(-1, kh, nq * g, d)
    table = s["table"].long()

    def rows(cache, scales):
        x = cache[table].float()
        if scales is not None:
            x = x * scales[table].transpose(-1, -2)[..., None]
        return x.flatten(1, 2)[:, :nk].permute(0, 2, 1, 3).contiguous()

    words = s["mask"].long()[at]  # [batch, nq, words]
    bits = (words[..., None] >> torch.arange(32, device="cuda") & 1).flatten(-2)
    bits = bits * (torch.arange(bits.shape[-1], device="cuda") < q_len[:, None, None])
    key = torch.arange(nk, device="cuda")
    base = (kv_len - q_len)[:, None, None]
    own_key = (key - base).clamp(0, bits.shape[-1] - 1).expand(-1, nq, -1)
    seen = torch.where(key < base, torch.ones_like(own_key), torch.gather(bits, 2, own_key)) > 0
    seen = seen & (key < kv_len[:, None, None])
    if c["window"]:
        seen = seen & ((key >= base) | (key > base + bits.sum(-1, keepdim=True) - 1 - c["window"]))
    seen = seen[:, None, :, None, :].expand(-1, 1, -1, g, -1).reshape(-1, 1, nq * g, nk)
    p = torch.matmul(q, rows(s["k"], s["sk"]).transpose(2, 3).contiguous())
    p.mul_(1.0 / math.sqrt(d)).masked_fill_(~seen, -math.inf)
    m = p.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, rows(s["v"], s["sv"])) / torch.where(total > 0, total, torch.ones_like(total))
    o = o.view(-1, kh, nq, g, d).permute(0, 2, 1, 3, 4).reshape(-1, nq, h, d)
    lse = (m + torch.log(total)).view(-1, kh, nq, g).permute(0, 2, 1, 3).reshape(-1, nq, h)
    token = torch.arange(s["tokens"], device="cuda")
    seq = torch.searchsorted(start[1:].contiguous(), token, right=True)
    i = token - start[seq]
    return dict(out=o[seq, i].to(s["q"].dtype), lse=lse[seq, i])


# ------------------------------------------------------------------------------------------
# The library's calls
# ------------------------------------------------------------------------------------------

def _ptr(t):
    return None if t is None else t.data_ptr()


def _space(lib, name, p, s):
    """The call's workspace, kept with the state as a program keeps it."""
    size = lib.op(name, "get_workspace_size")(ctypes.byref(p))
    s["workspace"] = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
    p.workspace, p.workspace_size = s["workspace"].data_ptr(), size


def _map(mod, s):
    c = s["case"]
    return mod.RopeMap(table=s["table"].data_ptr(), max_pos=c["max_pos"], rotary_dim=c["rot"],
                       interleaved=int(c["inter"]), inverse=0)


def _paged(mod, s):
    k, c = s["k"], s["case"]
    return mod.PagedKV(k=_ptr(k), v=_ptr(s["v"]), scale_k=_ptr(s["sk"]), scale_v=_ptr(s["sv"]),
                       num_pages=k.shape[-4], page_size=c["page"], kv_heads=c["kv_heads"], head_dim=c["dim"],
                       page_stride=k.stride(-4), token_stride=k.stride(-3), head_stride=k.stride(-2))


def _calls_norm(mod, lib, s):
    c = s["case"]
    d, row = c["dim"], c["heads"] * c["dim"]
    p = mod.NormRopeParams(
        rope=mod.RopeParams(tokens=c["tokens"], heads=c["heads"], head_dim=d, X=_ptr(s["x"]), x_token_stride=row,
                            x_head_stride=d, Y=_ptr(s["y"]), y_token_stride=row, y_head_stride=d,
                            positions=_ptr(s["pos"]), map=_map(mod, s)),
        norm=mod.HeadNorm(weight=_ptr(s["w"]), shift=c["shift"], eps=_EPS))
    calls, out = [(lib.op("norm_rope_" + c["type"], "run_async"), p)], dict(y=s["y"])
    if c["grad"]:
        q = mod.NormRopeGradParams(forward=p, dY=_ptr(s["dy"]), dy_token_stride=row, dy_head_stride=d,
                                   dX=_ptr(s["dx"]), dx_token_stride=row, dx_head_stride=d, dweight=_ptr(s["dw"]))
        _space(lib, "norm_rope_grad", q, s)
        calls.append((lib.op("norm_rope_grad_" + c["type"], "run_async"), q))
        out.update(dx=s["dx"], dw=s["dw"])
    return calls, lambda: out


def _calls_append(mod, lib, s):
    c = s["case"]
    h, kh, d, x = c["heads"], c["kv_heads"], c["dim"], s["qkv"]
    row, base, step = x.stride(0), x.data_ptr(), d * x.element_size()
    p = mod.KVAppendNormRopeParams(
        append=mod.KVAppendRopeParams(
            tokens=c["tokens"], K=base + h * step, k_token_stride=row, k_head_stride=d, V=base + (h + kh) * step,
            v_token_stride=row, v_head_stride=d, q_heads=h, Q=base, q_token_stride=row, q_head_stride=d,
            Q_out=_ptr(s["q_out"]), qo_token_stride=h * d, qo_head_stride=d, positions=_ptr(s["pos"]),
            slots=_ptr(s["slots"]), map=_map(mod, s), kv=_paged(mod, s)),
        q_norm=mod.HeadNorm(weight=_ptr(s["wq"]), shift=c["shift"], eps=_EPS),
        k_norm=mod.HeadNorm(weight=_ptr(s["wk"]), shift=c["shift"], eps=_EPS))
    name = "kv_append_norm_rope_%s_%s" % (c["cache"], c["src"])
    return [(lib.op(name, "run_async"), p)], lambda: _append_outputs(s)


def _calls_plan(mod, lib, s):
    c, out = s["case"], s["out"]
    p = mod.PagedPlanParams(
        batch=c["batch"], tokens=s["tokens"], page_size=c["page"], num_pages=s["pages"], block_table=_ptr(s["table"]),
        ld_table=s["table"].stride(0), free_pages=_ptr(s["free"]), free_capacity=s["free"].shape[0],
        ld_mask=s["words"] if c["tree"] else 0, **{k: _ptr(v) for k, v in out.items()},
        **{k: _ptr(s[k]) for k in ("new_len", "kv_len", "held", "free_count", "parent")})
    _space(lib, "paged_plan", p, s)
    got = dict(out, table=s["table"], free=s["free"])
    return [(lib.op("paged_plan", "run_async"), p)], lambda: got


def _calls_keep(mod, lib, s):
    c, scale = s["case"], s["sk"]
    p = mod.KVKeepParams(
        batch=c["batch"], max_keep=s["keep"].shape[1], q_start=_ptr(s["q_start"]), kv_len=_ptr(s["kv_len"]),
        kv_len_out=_ptr(s["kv_len_out"]), keep=_ptr(s["keep"]), ld_keep=s["keep"].stride(0),
        keep_len=_ptr(s["keep_len"]), block_table=_ptr(s["table"]), ld_table=s["table"].shape[1],
        layers=c["layers"], layer_stride=s["k"].stride(0), scale_layer_stride=0 if scale is None else scale.stride(0),
        kv=_paged(mod, s))
    return [(lib.op("kv_keep_" + c["cache"], "run_async"), p)], lambda: _keep_outputs(s, s["kv_len_out"])


def _calls_tree(mod, lib, s):
    c = s["case"]
    h, d = c["heads"], c["dim"]
    p = mod.AttnTreeParams(
        attn=mod.AttnPagedParams(
            batch=c["batch"], q_tokens=s["tokens"], q_heads=h, max_q_len=s["max_q"], max_kv_len=s["max_kv"],
            Q=_ptr(s["q"]), q_token_stride=h * d, q_head_stride=d, D=_ptr(s["out"]), d_token_stride=h * d,
            d_head_stride=d, lse=_ptr(s["lse"]), q_start=_ptr(s["q_start"]), kv_len=_ptr(s["kv_len"]),
            block_table=_ptr(s["table"]), ld_table=s["table"].shape[1], scale=1.0 / math.sqrt(d), causal=1,
            window=c["window"], kv=_paged(mod, s)),
        mask=_ptr(s["mask"]), ld_mask=s["mask"].stride(0))
    size = lib.op("attn_tree", "get_workspace_size")(ctypes.byref(p))
    s["workspace"] = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
    p.attn.workspace, p.attn.workspace_size = s["workspace"].data_ptr(), size
    out = dict(out=s["out"], lse=s["lse"])
    return [(lib.op("attn_tree_%s_%s" % (c["type"], c["cache"]), "run_async"), p)], lambda: out


def run(state):
    kind = state["case"]["kind"]
    if not own:
        return {"norm": _plain_norm, "append": _plain_append, "plan": _plain_plan, "keep": _plain_keep,
                "tree": _plain_tree}[kind](state)
    if "calls" not in state:  # entry points and their arguments, which a program builds once for its buffers
        build = {"norm": _calls_norm, "append": _calls_append, "plan": _calls_plan, "keep": _calls_keep,
                 "tree": _calls_tree}[kind]
        state["calls"] = build(*_tqt(), state)
    calls, outputs = state["calls"]
    stream = torch.cuda.current_stream().cuda_stream
    for f, p in calls:
        f(ctypes.byref(p), stream)
    return outputs()


# ------------------------------------------------------------------------------------------
# What a pass cannot do without
# ------------------------------------------------------------------------------------------

def _row_bytes(case):
    return case["dim"] + 4 if case["cache"] == "qsi8dx" else 2 * case["dim"]


def work(case):
    kind = case["kind"]
    if kind == "plan":
        s = [max(1, int(round(case["new"] * (1 - 0.7 * _spread(b))))) if case["tree"] or b % 3 else 1
             for b in range(case["batch"])]
        tokens = sum(s)
        per = 12 + (4 + 4 * -(-case["new"] // 32) if case["tree"] else 0)
        return dict(bytes=24 * case["batch"] + tokens * per + 8 * tokens // case["page"], flops=0)
    d = case["dim"]
    if kind == "norm":
        n = case["tokens"] * case["heads"] * d
        size = _SIZE[case["type"]]
        b = 2 * n * size + case["tokens"] * 4 * (case["rot"] + 1) + 4 * d
        f = 4 * n + 3 * case["tokens"] * case["heads"] * case["rot"]
        if case["grad"]:  # x and dy read, dx written
            b, f = b + 3 * n * size + 4 * d, 3 * f
        return dict(bytes=b, flops=f)
    kh = case["kv_heads"]
    if kind == "append":
        t, h, row = case["tokens"], case["heads"], _row_bytes(case)
        b = t * (h + 2 * kh) * d * _SIZE[case["src"]] + t * h * d * 2 + 2 * t * kh * row
        if case["cache"] == "qsi8dx":  # returned as the values it stands for
            b += 2 * case["slots"] * kh * (row + 2 * d)
        return dict(bytes=b + t * (4 * case["rot"] + 12), flops=t * (h + kh) * (4 * d + 3 * case["rot"]))
    row = 2 * kh * _row_bytes(case)
    if kind == "keep":
        most = min(case["accepted"], case["nodes"])
        moved = case["batch"] * case["layers"] * (most - 1) / 2
        b = 2 * moved * row + case["batch"] * 4 * (most + 4)
        if case["cache"] == "qsi8dx":
            b += case["batch"] * case["layers"] * case["kv"] * (row + 4 * kh * d)
        return dict(bytes=b, flops=0)
    lengths = _lengths(case)
    tokens, pairs, keys = 0, 0, 0
    for n, kv in lengths:
        seen = min(kv - n, case["window"] or kv)
        tokens += n
        keys += seen + n
        pairs += n * seen + n * min(n, 4)  # of its own tree a token sees the path to it
    return dict(bytes=tokens * case["heads"] * (4 * d + 4) + row * keys, flops=4 * d * case["heads"] * pairs)


# ------------------------------------------------------------------------------------------
# The same results in 64 bits
# ------------------------------------------------------------------------------------------

def _exact_turn(x, case, s):
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
    return torch.cat((z.reshape(*x.shape[:2], r), x[..., r:]), -1)


def _exact_norm_rows(x, w, case):
    length = torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + _EPS)
    return x / length * (w + case["shift"])


def _exact_norm(case, s):
    x = s["x"].double().requires_grad_(case["grad"])
    w = s["w"].double().requires_grad_(case["grad"])
    y = _exact_turn(_exact_norm_rows(x, w, case), case, s)
    out = dict(y=y.detach())
    if case["grad"]:
        out["dx"], out["dw"] = torch.autograd.grad(y, (x, w), s["dy"].double())
    return out


def _exact_append(case, s):
    h, kh, page = case["heads"], case["kv_heads"], case["page"]
    x = s["qkv"].double()
    q = _exact_turn(_exact_norm_rows(x[:, :h], s["wq"].double(), case), case, s)
    k = _exact_turn(_exact_norm_rows(x[:, h:h + kh], s["wk"].double(), case), case, s)
    out = dict(q=q)
    for name, scale, rows in (("k", "sk", k), ("v", "sv", x[:, h + kh:])):
        old = s[name].double()
        if s[scale] is not None:
            old = old * s[scale].double().permute(0, 2, 1).unsqueeze(-1)
            step = rows.abs().max(-1, keepdim=True).values / 127
            rows = torch.where(step > 0, torch.round(rows / step) * step, torch.zeros_like(rows))
        old[s["slots"] // page, s["slots"] % page] = rows
        out[name] = old
    return out


def _exact_keep(case, s):
    page, out = case["page"], {}
    starts, lens = s["q_start"].tolist(), s["kv_len"].tolist()
    keep, n = s["keep"].tolist(), s["keep_len"].tolist()
    table = s["table"].tolist()
    src, dst, kv_len = [], [], []
    for b in range(case["batch"]):
        base = lens[b] - (starts[b + 1] - starts[b])
        for j in range(n[b]):
            at, to = base + keep[b][j], base + j
            src.append(table[b][at // page] * page + at % page)
            dst.append(table[b][to // page] * page + to % page)
        kv_len.append(base + n[b])
    src, dst = _ints(src, torch.int64), _ints(dst, torch.int64)
    for name, scale in (("k", "sk"), ("v", "sv")):
        x = s[name].double()
        if s[scale] is not None:
            x = x * s[scale].double().transpose(-1, -2).unsqueeze(-1)
        x = x.flatten(1, 2)
        x[:, dst] = x[:, src].clone()
        out[name] = x.view(s[name].shape)
    return dict(out, kv_len=_ints(kv_len))


def _exact_tree(case, s):
    h, kh, d = case["heads"], case["kv_heads"], case["dim"]
    out = torch.zeros((s["tokens"], h, d), dtype=torch.float64, device="cuda")
    lse = torch.zeros((s["tokens"], h), dtype=torch.float64, device="cuda")
    words = s["mask"].cpu().numpy().view("uint32").tolist()
    first = 0
    for b, (nq, nk) in enumerate(_lengths(case)):
        pages = s["table"][b, :-(-nk // case["page"])].long()
        rows = [sum(w << (32 * i) for i, w in enumerate(words[first + t])) for t in range(nq)]
        hidden = torch.zeros((nq, nk), dtype=torch.bool)
        for t, bits in enumerate(rows):
            depth = bin(bits & ((1 << nq) - 1)).count("1")
            if case["window"]:
                hidden[t, :max(0, min(nk - nq, nk - nq + depth - case["window"]))] = True
            hidden[t, nk - nq:] = torch.tensor([not (bits >> u) & 1 for u in range(nq)])
        hidden = hidden.cuda()
        for j in range(kh):
            kv = []
            for name, scale in (("k", "sk"), ("v", "sv")):
                rows = s[name][pages, :, j].double()
                if s[scale] is not None:
                    rows = rows * s[scale][pages, j].double()[..., None]
                kv.append(rows.reshape(-1, d)[:nk])
            for i in range(j * (h // kh), (j + 1) * (h // kh)):
                a = (s["q"][first:first + nq, i].double() @ kv[0].T) / math.sqrt(d)
                a[hidden] = -math.inf
                out[first:first + nq, i] = torch.softmax(a, -1) @ kv[1]
                lse[first:first + nq, i] = torch.logsumexp(a, -1)
        first += nq
    return dict(out=out, lse=lse)


def exact(case, seed):
    if case["kind"] == "plan":  # whole numbers
        return None
    s = prepare(case, seed)
    return {"norm": _exact_norm, "append": _exact_append, "keep": _exact_keep,
            "tree": _exact_tree}[case["kind"]](case, s)
