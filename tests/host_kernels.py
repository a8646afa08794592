"""The kernels of the steps with drafted tokens and of the paged attention on the CPU (test infrastructure): their sources,
with tests/host_hip.hpp in the place of HIP, behind the library's own entry points. Arrays lie against pages that no access
may touch, so that a read or write out of range ends the process, which tests/test_kernels_on_host.py starts for that."""

import concurrent.futures
import ctypes
import ctypes.util
import glob
import mmap
import os
import re
import subprocess

import numpy as np

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "torq-tile_amd", "csrc")
CLANG = "/opt/rocm/llvm/bin/clang++"
SOURCES = ["attn_paged_f16", "attn_tree_f16", "paged_plan", "kv_keep", "norm_rope"]
# What the CPU has no instruction for: (file, pattern, replacement); each pattern is there once at least.
PATCHES = [
    ("attn_common.hpp", r"float y = x;\n#if defined\(__HIP_DEVICE_COMPILE__\)\n.*?#endif\n    return fmaxf\(x, y\);",
     "return host_hip::max_across_halves(x);"),
    ("attn_common.hpp", r"typedef __attribute__\(\(address_space\(3\)\)\) i16x4 lds_i16x4;\n.*?;\n",
     "return __builtin_bit_cast(u32x2, host_read_column4(p));\n"),
    # (on the GPU it reads a lane that does not take part)
    ("attn_common.hpp", r"return lane < n \? x : __builtin_amdgcn_readlane\(x, n - 1\);",
     "const int last = __builtin_amdgcn_readlane(x, n - 1);\n    return lane < n ? x : last;"),
    ("attn_tile.hpp", r'asm volatile\("s_waitcnt vmcnt\(0\)" ::: "memory"\);', "host_hip::wait_loads();"),
    ("attn_tile.hpp", r'asm volatile\("" : [^;]*\);', ""),
]


def build(folder):
    """The library, in `folder`."""
    for path in glob.glob(os.path.join(CSRC, "*.hpp")) + [os.path.join(CSRC, s + ".hip") for s in SOURCES]:
        name = os.path.basename(path)
        with open(path) as f:
            text = f.read()
        for file, pattern, by in PATCHES:
            if file == name:
                text, n = re.subn(pattern, lambda m, by=by: by, text, flags=re.S if "\n" in pattern or ".*?" in pattern else 0)
                assert n > 0, (file, pattern)
        assert not re.search(r"\basm\b\s*(volatile)?\s*\(", text) or not name.startswith("attn_"), name
        with open(os.path.join(folder, name), "w") as f:
            f.write(text)
    with open(os.path.join(ROOT, "tests", "host_hip.hpp")) as f, \
            open(os.path.join(folder, "tqt_hip_common.hpp"), "w") as g:
        g.write(f.read())
    flags = ["-std=c++17", "-O1", "-march=x86-64-v3", "-fPIC", "-ffp-contract=off", "-w",
             "-I" + os.path.join(ROOT, "include")]

    def compiled(s):
        out = os.path.join(folder, s + ".o")
        subprocess.run([CLANG, "-x", "c++", *flags, "-c", os.path.join(folder, s + ".hip"), "-o", out], check=True)
        return out

    with concurrent.futures.ThreadPoolExecutor(len(SOURCES)) as pool:
        objects = list(pool.map(compiled, SOURCES))
    out = os.path.join(folder, "libkernels_on_host.so")
    subprocess.run([CLANG, "-shared", "-o", out, *objects], check=True)
    return out


_LIBC = ctypes.CDLL(None, use_errno=True)
_LIBC.mmap.restype = ctypes.c_void_p
_LIBC.mmap.argtypes = [ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_long]
_LIBC.mprotect.argtypes = [ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int]
_LIBC.munmap.argtypes = [ctypes.c_void_p, ctypes.c_size_t]
PAGE = mmap.PAGESIZE


class Arena:
    """Arrays between pages that may not be touched, against the one behind them, or with `low` the one before."""

    def __init__(self, low=False):
        self.low, self.maps = low, []

    def put(self, a):
        a = np.ascontiguousarray(a)
        size = -(-max(a.nbytes, 1) // PAGE) * PAGE
        at = _LIBC.mmap(None, size + 2 * PAGE, mmap.PROT_READ | mmap.PROT_WRITE,
                        mmap.MAP_PRIVATE | mmap.MAP_ANONYMOUS, -1, 0)
        assert at not in (None, ctypes.c_void_p(-1).value)
        assert _LIBC.mprotect(at, PAGE, 0) == 0 and _LIBC.mprotect(at + PAGE + size, PAGE, 0) == 0
        self.maps.append((at, size + 2 * PAGE))
        start = at + PAGE + (0 if self.low else size - a.nbytes)
        got = np.frombuffer((ctypes.c_char * a.nbytes).from_address(start), a.dtype).reshape(a.shape) if a.nbytes else a
        if a.nbytes:
            got[...] = a
        return got

    def close(self):
        for at, size in self.maps:
            _LIBC.munmap(at, size)
        self.maps = []


def ptr(a):
    return None if a is None else a.ctypes.data


class Library:
    """The entry points, as tqt_testlib's library gives them."""

    def __init__(self, path):
        self.dll = ctypes.CDLL(path)

    def call(self, name, p):
        error = getattr(self.dll, "tqt_get_error_%s_gfx950" % name)
        error.restype = ctypes.c_char_p
        why = error(ctypes.byref(p))
        assert why is None, (name, why)
        getattr(self.dll, "tqt_run_%s_gfx950" % name)(ctypes.byref(p))

    def workspace(self, name, p, at, arena):
        f = getattr(self.dll, "tqt_get_workspace_size_%s_gfx950" % name)
        f.restype = ctypes.c_size_t
        size = f(ctypes.byref(p))
        space = arena.put(np.full(-(-size // 16) * 4, np.nan, np.float32))
        at.workspace, at.workspace_size = (ptr(space) if size else None), size
        return space


# ------------------------------------------------------------------------------------------
# Random calls, each against its plain form
# ------------------------------------------------------------------------------------------

def structs():
    import importlib.util

    spec = importlib.util.spec_from_file_location("tqt_gfx950", os.path.join(ROOT, "torq-tile_amd", "tqt_gfx950.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def cache_of(mod, arena, rng, quant, pages, page, kv_heads, d, heads_first):
    """A cache's struct, its arrays, and k and v [pages, page, heads, d] as numbers."""
    arrays, values = [], []
    for _ in range(2):
        if quant:
            x = rng.integers(-127, 128, (pages, page, kv_heads, d)).astype(np.int8)
            s = (rng.random((pages, kv_heads, page)) * 0.02 + 0.003).astype(np.float32)
            values.append(x * s.astype(np.float64).transpose(0, 2, 1)[..., None])
        else:
            x, s = rng.standard_normal((pages, page, kv_heads, d)).astype(np.float16), None
            values.append(x.astype(np.float64))
        arrays.append((arena.put(x.transpose(0, 2, 1, 3) if heads_first else x), None if s is None else arena.put(s)))
    (k, sk), (v, sv) = arrays
    kv = mod.PagedKV(k=ptr(k), v=ptr(v), scale_k=ptr(sk), scale_v=ptr(sv), num_pages=pages, page_size=page,
                     kv_heads=kv_heads, head_dim=d, page_stride=page * kv_heads * d,
                     token_stride=d if heads_first else kv_heads * d, head_stride=page * d if heads_first else d)
    return kv, arrays, values


def attention(lib, mod, rng, arena, tree, cache, lengths, heads, kv_heads, d, page, window=0, words=None, max_q=None,
              max_kv=None, more_rows=0, holes=0.0, causal=True):
    """One call over lengths (new tokens, keys); its workspace size."""
    import drafted_ref as D
    import paged_ref as R

    batch, starts = len(lengths), np.concatenate(([0], np.cumsum([q for q, _ in lengths]))).astype(np.int32)
    max_q = max(q for q, _ in lengths) if max_q is None else max_q
    max_kv = max(n for _, n in lengths) if max_kv is None else max_kv
    ld = -(-max_kv // page)
    pages = max(1, sum(-(-n // page) for _, n in lengths))
    order, at = rng.permutation(pages), 0
    table = rng.choice([-1, pages, 2 ** 31 - 1, -2 ** 31], (batch, ld)).astype(np.int32)
    for b, (_, n) in enumerate(lengths):
        m = min(-(-n // page), ld)
        table[b, :m] = order[at:at + m]
        at += m
    gone = rng.random((batch, ld)) < holes
    table[gone] = rng.choice([-1, pages, 2 ** 31 - 1, -2 ** 31], int(gone.sum()))
    rows = int(starts[-1]) + more_rows
    q = (rng.standard_normal((rows, heads, d)) * 1.5).astype(np.float16)
    heads_first = bool(rng.integers(0, 2))
    kv, _, (k, v) = cache_of(mod, arena, rng, cache == "qsi8dx", pages, page, kv_heads, d, heads_first)
    dq, out = arena.put(q), arena.put(np.full(q.shape, 9, np.float16))
    lse = arena.put(np.full((rows, heads), 9, np.float32))
    ints = [arena.put(x) for x in (starts, np.array([n for _, n in lengths], np.int32), table)]
    p = mod.AttnPagedParams(
        batch=batch, q_tokens=rows, q_heads=heads, max_q_len=max_q, max_kv_len=max_kv, Q=ptr(dq),
        q_token_stride=heads * d, q_head_stride=d, D=ptr(out), d_token_stride=heads * d, d_head_stride=d, lse=ptr(lse),
        q_start=ptr(ints[0]), kv_len=ptr(ints[1]), block_table=ptr(ints[2]), ld_table=ld, scale=d ** -0.5,
        causal=int(causal), window=window, kv=kv)
    see = []
    if tree:
        words = -(-max(max_q, 1) // 32) if words is None else words
        mask = np.zeros((rows, words), np.uint32)
        for b, (nq, _) in enumerate(lengths):
            parents = D.random_parents(rng, nq, 0.5)
            mask[starts[b]:starts[b + 1]] = D.pack([D.path(parents, i) for i in range(nq)], words)
        mask[starts[-1]:] = 0xffffffff
        masks = arena.put(mask)
        call = mod.AttnTreeParams(attn=p, mask=ptr(masks), ld_mask=words)
        name, base = "attn_tree", call.attn
    else:
        call, name, base = p, "attn_paged", p
    space = lib.workspace(name, call, base, arena)
    lib.call("%s_f16_%s" % (name, cache), call)
    for b, (nq, nk) in enumerate(lengths):
        lo, n = int(starts[b]), min(nq, max_q)
        if nk > max_kv:
            continue
        j = np.arange(nk)
        page_of = table[b, j // page].astype(np.int64)
        kept = (page_of >= 0) & (page_of < pages)
        page_of = np.where(kept, page_of, 0)
        see = (D.visible_tree(mask[lo:lo + nq], nq, nk, window) if tree else R.visible(nq, nk, causal, window)) & kept
        want = R.attention(q[lo:lo + n].astype(np.float64), k[page_of, j % page], v[page_of, j % page], see[:n], d ** -0.5)
        tol, tol_lse = R.attention_bound("f16", d, *want)
        off = np.abs(out[lo:lo + n] - want[0])
        assert (off <= tol).all(), (b, nq, nk, np.nanmax(off / tol))
        none = np.isneginf(want[1])
        np.testing.assert_array_equal(np.isneginf(lse[lo:lo + n]), none)
        with np.errstate(invalid="ignore"):
            assert (np.abs(lse[lo:lo + n] - want[1])[~none] <= tol_lse[~none]).all()
        assert (out[lo + n:lo + nq] == 9).all()
    assert (out[starts[-1]:] == 9).all() and (lse[starts[-1]:] == 9).all()
    return base.workspace_size


def suite_attention(lib, mod, seed, cases=40):
    """Few rows, tiles, both; splits and joins; windows, pages that are not kept, bounds above and below the lengths."""
    rng = np.random.default_rng(seed)
    split = 0
    for case in range(cases):
        arena = Arena(low=bool(case & 1))
        tree, cache = bool(rng.random() < 0.7), ["f16", "qsi8dx"][int(rng.integers(0, 2))]
        d = int(rng.choice([16, 48, 64, 64, 80, 128, 144, 256]))
        kv_heads, group = int(rng.integers(1, 4)), int(rng.choice([1, 2, 4, 5]))
        batch = int(rng.integers(1, 4)) if rng.random() < 0.9 else 66
        most_q = int(rng.choice([1, 3, 8, 33, 70])) if batch < 66 else 2
        most_kv = int(rng.choice([20, 130, 400])) if batch < 66 else 40
        lengths = [(int(rng.integers(0, most_q + 1)), int(rng.integers(0, most_kv + 1))) for _ in range(batch)]
        lengths[-1] = (most_q, most_kv)
        kw = dict(page=int(rng.choice([1, 3, 16, 24, 64])), window=int(rng.choice([0, 0, 0, 1, 37, 2 ** 31 - 1])),
                  holes=float(rng.choice([0, 0.2])), more_rows=int(rng.integers(0, 3)))
        if rng.random() < 0.3:
            kw["max_kv"] = most_kv + int(rng.integers(0, 5000))
        if rng.random() < 0.2:
            kw["max_kv"] = max(1, most_kv // 2)
        if rng.random() < 0.2:
            kw["max_q"] = max(1, most_q // 2)
        elif rng.random() < 0.2:
            kw["max_q"] = most_q + int(rng.integers(0, 60))
        if tree and rng.random() < 0.3:
            kw["words"] = -(-kw.get("max_q", most_q) // 32) + 2
        print("attention", seed, case, tree, cache, lengths[:4], batch, group * kv_heads, kv_heads, d, kw, flush=True)
        split += attention(lib, mod, rng, arena, tree, cache, lengths, group * kv_heads, kv_heads, d, **kw) > 0
        arena.close()
    assert split > cases // 8


def suite_spans(lib, mod, seed):
    """Tiles of trees in equal spans of each sequence's own: what the grid and the workspace hold, as the kernel and the
    join find it. The bounds are above the lengths, as a program's are."""
    rng = np.random.default_rng(seed)
    ragged = [(40, 700), (33, 130), (64, 520), (20, 64), (17, 17), (50, 300), (5, 90), (0, 30), (21, 0)]
    for case, (lengths, max_kv, window) in enumerate((
            (ragged, 2000, 0), ([(17 + 5 * i, 40 + 171 * i) for i in range(9)], 6000, 1200),
            ([(int(rng.integers(0, 65)), int(rng.integers(0, 400))) for _ in range(8)] + [(64, 900)], 1900, 0),
            ([(60, 300)] * 10, 2500, 0))):
        arena = Arena(low=bool(case & 1))
        cache = ["f16", "qsi8dx"][case & 1]
        print("spans", seed, case, cache, lengths, flush=True)
        size = attention(lib, mod, rng, arena, True, cache, lengths, 16, 8, 64, 16, max_kv=max_kv, window=window)
        assert size > 0
        arena.close()


def suite_plan(lib, mod, seed, cases=60):
    import drafted_ref as D

    rng = np.random.default_rng(seed)
    for case in range(cases):
        arena = Arena(low=bool(case & 1))
        batch = int(rng.choice([1, 3, 20, 70, 1030])) if case % 10 else 1030
        most, page = int(rng.choice([1, 9, 40])), int(rng.choice([1, 4, 16, 100]))
        new = rng.integers(0, most + 1, batch)
        new[rng.random(batch) < 0.2] = -1
        kv = rng.integers(0, 90, batch)
        own = -(-kv // page)
        held = own + rng.integers(0, 3, batch)
        ld = int(rng.integers(max(1, own.max()), own.max() + 40 // page + 3))
        held = np.minimum(held, ld)
        used = int(held.sum())
        spare = int(rng.integers(0, batch * 3 + 2))
        pages = used + spare + 1
        order, at = rng.permutation(pages), 0
        table = np.full((batch, ld), -7, np.int32)
        for b in range(batch):
            table[b, :held[b]] = order[at:at + held[b]]
            at += held[b]
        holes = rng.random(table.shape) < 0.02
        table[holes] = rng.choice([-1, pages, 2 ** 31 - 1], int(holes.sum()))
        free = np.full(pages, -9, np.int32)
        free[:spare] = order[at:at + spare]
        tokens = max(0, int(np.maximum(new, 0).sum()) + int(rng.integers(-3, 5)))
        parent, words = None, 0
        if rng.random() < 0.6:
            words = int(rng.integers(1, 4))
            parent = np.array([int(rng.integers(-2, 60)) for _ in range(tokens)], np.int32)
        print("plan", seed, case, batch, tokens, page, ld, words, flush=True)
        want = D.plan(new, kv, held, table, free, spare, tokens, page, pages, parent, words)
        a = {k: arena.put(np.asarray(x, np.int32)) for k, x in (
            ("new_len", new), ("kv_len", kv), ("held", held), ("block_table", table), ("free_pages", free),
            ("free_count", [spare]))}
        out = {k: arena.put(np.full(n, 77, np.int32)) for k, n in (
            ("kv_len_out", batch), ("held_out", batch), ("free_count_out", 1), ("refused", 1), ("q_start", batch + 1),
            ("positions", tokens))}
        out["slots"] = arena.put(np.full(tokens, 77, np.int64))
        if rng.random() < 0.5:
            out.update(kv_len_out=a["kv_len"], held_out=a["held"], free_count_out=a["free_count"])
        if parent is not None:
            a["parent"], out["mask"] = arena.put(parent), arena.put(np.zeros((tokens, words), np.int32))
        p = mod.PagedPlanParams(batch=batch, tokens=tokens, page_size=page, num_pages=pages, ld_table=ld,
                                free_capacity=pages, ld_mask=words, **{k: ptr(x) for k, x in {**a, **out}.items()})
        if parent is not None and tokens == 0:
            p.parent = p.mask = 16  # not read
        space = lib.workspace("paged_plan", p, p, arena)
        lib.call("paged_plan", p)
        for k, x in out.items():
            np.testing.assert_array_equal(x.view(np.uint32) if k == "mask" else x, want[k], k)
        np.testing.assert_array_equal(a["block_table"], want["table"])
        np.testing.assert_array_equal(a["free_pages"], want["free"])
        arena.close()


def suite_keep(lib, mod, seed, cases=60):
    import drafted_ref as D

    rng = np.random.default_rng(seed)
    for case in range(cases):
        arena = Arena(low=bool(case & 1))
        quant, d, kv_heads = bool(rng.integers(0, 2)), int(rng.choice([16, 48, 64])), int(rng.integers(1, 4))
        batch, page, layers = int(rng.integers(1, 6)), int(rng.choice([1, 4, 16])), 1
        lengths = [(int(rng.integers(0, 30)), int(rng.integers(0, 80))) for _ in range(batch)]
        ld = max(1, max(-(-n // page) for _, n in lengths))
        pages = batch * ld
        table = rng.permutation(pages).reshape(batch, ld).astype(np.int32)
        holes = rng.random(table.shape) < 0.1
        table[holes] = rng.choice([-1, pages, 2 ** 31 - 1, -2 ** 31], int(holes.sum()))
        keep = np.sort(rng.integers(-1, 32, (batch, 9)), 1).astype(np.int32)
        count = rng.integers(-2, 12, batch).astype(np.int32)
        most = int(rng.integers(0, 10))
        starts = np.concatenate(([0], np.cumsum([n for n, _ in lengths]))).astype(np.int32)
        tokens = int(starts[-1])
        served = rng.random(batch) < 0.7
        kv, arrays, _ = cache_of(mod, arena, rng, quant, pages, page, kv_heads, d, False)
        before = [[None if x is None else x.copy() for x in pair] for pair in arrays]
        kv_len = arena.put(np.array([n for _, n in lengths], np.int32))
        positions = np.concatenate([np.full(q, n - q if ok else n) for (q, n), ok in zip(lengths, served)] + [[]])
        positions = arena.put(positions.astype(np.int32))
        out, ints = arena.put(np.full(batch, 77, np.int32)), [arena.put(x) for x in (starts, keep, count, table)]
        p = mod.KVKeepParams(
            batch=batch, max_keep=most, q_start=ptr(ints[0]), kv_len=ptr(kv_len), kv_len_out=ptr(out), keep=ptr(ints[1]),
            ld_keep=9, keep_len=ptr(ints[2]), block_table=ptr(ints[3]), ld_table=ld, layers=layers, kv=kv,
            positions=ptr(positions) if tokens else None, tokens=tokens)
        print("keep", seed, case, quant, d, kv_heads, page, lengths, flush=True)
        lib.call("kv_keep_" + ("qsi8dx" if quant else "f16"), p)
        for b, (nq, n) in enumerate(lengths):
            if nq and (not served[b] or n - nq >= n):
                assert out[b] == n
                continue
            if n < nq:
                # its first position, n - nq, is below its length
                assert out[b] == 0
                continue
            path = D.kept(keep[b], count[b], nq, most)
            assert out[b] == n - nq + len(path)
            for j, i in enumerate(path):
                (ps, os_), (pd, od) = (divmod(n - nq + x, page) for x in (i, j))
                ps, pd = int(table[b, ps]), int(table[b, pd])
                if 0 <= ps < pages and 0 <= pd < pages:
                    for (x, s), (x0, s0) in zip(arrays, before):
                        assert (x[pd, od] == x0[ps, os_]).all()
                        assert s is None or (s[pd, :, od] == s0[ps, :, os_]).all()
        arena.close()


def suite_norm(lib, mod, seed, cases=40):
    import drafted_ref as D
    import paged_ref as R

    rng = np.random.default_rng(seed)
    for case in range(cases):
        arena = Arena(low=bool(case & 1))
        kind = ["f32", "f16"][int(rng.integers(0, 2))]
        t = np.float32 if kind == "f32" else np.float16
        d = int(rng.choice([16, 48, 64, 80, 128, 10, 7, 130, 1040]))
        rot = int(rng.choice([d // 2 * 2, d // 4 * 2, 0]))
        tokens, heads = int(rng.integers(1, 30)), int(rng.integers(1, 6))
        inter, shift = bool(rng.integers(0, 2)), float(rng.integers(0, 2))
        x, dy = (arena.put((rng.standard_normal((tokens, heads, d)) * 2).astype(t)) for _ in range(2))
        y, dx = (arena.put(np.full(x.shape, 9, t)) for _ in range(2))
        w = arena.put((rng.standard_normal(d) * 0.3 + 1 - shift).astype(np.float32))
        dw = arena.put(np.full(d, 9, np.float32))
        table = arena.put(R.rope_table(50, rot).astype(np.float32)) if rot else None
        pos = arena.put(rng.integers(0, 50, tokens).astype(np.int32))
        p = mod.NormRopeParams(
            rope=mod.RopeParams(tokens=tokens, heads=heads, head_dim=d, X=ptr(x), x_token_stride=heads * d,
                                x_head_stride=d, Y=ptr(y), y_token_stride=heads * d, y_head_stride=d,
                                positions=ptr(pos), map=mod.RopeMap(table=ptr(table), max_pos=50 if rot else 0,
                                                                    rotary_dim=rot, interleaved=int(inter))),
            norm=mod.HeadNorm(weight=ptr(w), shift=shift, eps=1e-5))
        print("norm", seed, case, kind, tokens, heads, d, rot, inter, flush=True)
        lib.call("norm_rope_" + kind, p)
        g = mod.NormRopeGradParams(forward=p, dY=ptr(dy), dy_token_stride=heads * d, dy_head_stride=d, dX=ptr(dx),
                                   dx_token_stride=heads * d, dx_head_stride=d, dweight=ptr(dw))
        space = lib.workspace("norm_rope_grad", g, g, arena)
        lib.call("norm_rope_grad_" + kind, g)
        u, tiny = R.ROUND[kind]
        args = (pos, table, rot, inter, w, shift, 1e-5)
        x, dy = x.astype(np.float64), dy.astype(np.float64)
        want, tol = D.norm_rope(x, *args)
        assert (np.abs(y - want) <= tol + (np.abs(want) + tol) * u * 1.01 + tiny).all()
        want, want_w, tol, tol_w = D.norm_rope_grad(x, dy, *args, 1)
        assert (np.abs(dx - want) <= tol + (np.abs(want) + tol) * u * 1.01 + tiny).all()
        assert (np.abs(dw - want_w) <= tol_w).all()
        arena.close()


if __name__ == "__main__":
    import sys

    globals()["suite_" + sys.argv[2]](Library(sys.argv[1]), structs(), int(sys.argv[3]))
    print("whole")
