"""Plain forms of the operators of a serving step with drafted tokens: the norm of heads with its rotation and the
gradient, a step's plan, kept rows, tree masks (test infrastructure, numpy only; the builders take torch tensors)."""

import ctypes

import numpy as np

import paged_ref as R


# ------------------------------------------------------------------------------------------
# The norm of heads, with rotation
# ------------------------------------------------------------------------------------------

def normed(x, weight, shift, eps):
    """x [tokens, heads, d] f64."""
    n = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    return n if weight is None else n * (weight.astype(np.float64) + shift)


def norm_rope(x, pos, table, rot, inter, weight, shift, eps, inverse=False):
    """The result in 64 bits, and how far the f32 steps may be from it: r is rounded once (its sum is in 64 bits), x r,
    weight + shift and their product once each, so a normalised value is off by 4 half steps; the rotation
    rounds each product and the sum."""
    n = normed(x, weight, shift, eps)
    y, size = R.rope(n, pos, table, rot, inter, inverse)
    return y, size * (4 * 2.0 ** -24 + 2 * 2.0 ** -24) * 1.01


def norm_rope_grad(x, dy, pos, table, rot, inter, weight, shift, eps, rows_in_f32, inverse=False):
    """dx, dweight, and their bounds (before the rounding to dx's type). rows_in_f32: rows that a thread adds up
    in f32."""
    d = x.shape[-1]
    u, su = R.rope(dy, pos, table, rot, inter, not inverse)
    f = np.ones(d) if weight is None else weight.astype(np.float64) + shift
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    m = x * r
    mean = (f * u * m).mean(-1, keepdims=True)
    dx = r * (f * u - m * mean)
    # of the terms' size: u 2 half steps, f 1, their product 1; the mean 5 (u, f, product, its rounding), m 2, their
    # product 1; the difference 1, r 1 and the last product 1: 11 at most
    terms = r * (np.abs(f) * su + np.abs(m) * (np.abs(f) * su * np.abs(m)).mean(-1, keepdims=True))
    dw = (u * m).sum((0, 1))
    # a term: u 2, m 2, their product 1; a sum of k terms k - 1; the shares' and the result's rounding
    dw_tol = (su * np.abs(m)).sum((0, 1)) * (5 + rows_in_f32 + 2) * 2.0 ** -24 * 1.01
    return dx, dw, terms * 12 * 2.0 ** -24, dw_tol + 1e-30


# ------------------------------------------------------------------------------------------
# Trees
# ------------------------------------------------------------------------------------------

def random_parents(rng, n, chain=0.0):
    """parent of every token among n: an earlier one, or -1; now and then the one before."""
    p = np.array([int(rng.integers(-1, i)) if i else -1 for i in range(n)], np.int32)
    back = rng.random(n) < chain
    p[back] = np.arange(n)[back] - 1
    return p


def path(parents, i):
    """Token i and those that it descends from."""
    got = []
    while i >= 0:
        got.append(i)
        i = int(parents[i]) if -1 <= parents[i] < i else -1
    return got


def pack(rows, words):
    """rows: sets of bits, as [len(rows), words] uint32."""
    out = np.zeros((len(rows), words), np.uint32)
    for i, bits in enumerate(rows):
        for t in bits:
            if t < 32 * words:
                out[i, t // 32] |= np.uint32(1 << (t % 32))
    return out


def visible_tree(mask, nq, nk, window):
    """[nq, nk] from nq mask rows, as the operator defines it."""
    base = nk - nq
    see = np.zeros((nq, nk), bool)
    for i in range(nq):
        bits = [t for t in range(min(nq, 32 * mask.shape[1])) if mask[i, t // 32] >> (t % 32) & 1]
        for j in range(nk):
            if j < base:
                see[i, j] = not window or j > base + len(bits) - 1 - window
        for t in bits:
            if 0 <= base + t < nk:
                see[i, base + t] = True
    return see


# ------------------------------------------------------------------------------------------
# A step's plan and kept rows
# ------------------------------------------------------------------------------------------

def plan(new_len, kv_len, held, table, free, count, tokens, page, num_pages, parent=None, words=0):
    """What tqt_run_paged_plan writes, step by step as its header says."""
    batch, ld = table.shape
    table, free = table.copy(), free.copy()
    kv_len = np.clip(kv_len.astype(np.int64), 0, 2 ** 30)
    pages_of = lambda n: -(-n // page)  # noqa: E731
    kv_out, held_out = kv_len.copy(), np.zeros(batch, np.int64)
    count = min(max(int(count), 0), len(free))
    for b in range(batch):
        if new_len[b] < 0:
            for j in range(min(max(int(held[b]), 0), ld)):
                if 0 <= table[b, j] < num_pages:
                    if count < len(free):
                        free[count] = table[b, j]
                    count += 1
            kv_out[b] = 0
    top = min(count, len(free))
    start, starts, total, needed, refused, seqs = 0, [], 0, 0, 0, []
    taken = 0
    for b in range(batch):
        n = min(max(int(new_len[b]), 0), 2 ** 30)
        total += n
        starts.append(min(start, tokens))
        start += n
        own = pages_of(int(kv_len[b]))
        h = max(min(max(int(held[b]), 0), ld), own)
        served = False
        if new_len[b] >= 0:
            need = max(pages_of(int(kv_len[b]) + n) - h, 0)
            fits = (n == 0 or total <= tokens) and h + need <= ld and kv_len[b] + n <= 2 ** 30
            need = need if fits else 0
            served = fits and (need == 0 or needed + need <= top)
            needed += need
            held_out[b] = h
            if served:
                for j in range(need):
                    table[b, h + j] = free[top - 1 - taken - j]
                taken += need
                held_out[b] += need
                kv_out[b] += n
            else:
                refused += 1
        seqs.append((n, served))
    starts.append(min(start, tokens))
    positions, slots = np.zeros(tokens, np.int64), np.full(tokens, -1, np.int64)
    mask = np.zeros((tokens, words), np.uint32)
    for b, (n, served) in enumerate(seqs):
        lo, hi = starts[b], starts[b + 1]
        for i in range(hi - lo):
            at = int(kv_len[b]) + i
            positions[lo + i] = at
            if parent is not None:
                up = path(parent[lo:hi], i)
                positions[lo + i] = int(kv_len[b]) + len(up) - 1
                mask[lo + i] = pack([up], words)[0]
            if served and 0 <= table[b, at // page] < num_pages:
                slots[lo + i] = int(table[b, at // page]) * page + at % page
    return dict(kv_len_out=kv_out, held_out=held_out, free_count_out=np.array([top - taken]),
                refused=np.array([refused]), q_start=np.array(starts), positions=positions, slots=slots,
                table=table, free=free, mask=mask)


def kept(keep, n, q_len, max_keep):
    """The entries of a list that count."""
    got = []
    for x in keep[:min(max(int(n), 0), max_keep)]:
        if not (got[-1] if got else -1) < x < q_len:
            break
        got.append(int(x))
    return got


# ------------------------------------------------------------------------------------------
# Calls
# ------------------------------------------------------------------------------------------

def head_norm(mod, weight, shift, eps):
    return mod.HeadNorm(weight=R.ptr(weight), shift=shift, eps=eps)


def workspace(lib, name, p, at=None):
    """Gives a call its workspace, filled with NaN; `at`: the struct that holds the fields."""
    import torch

    size = lib.op(name, "get_workspace_size")(ctypes.byref(p))
    space = torch.full((max(size // 4, 4) + 64,), float("nan"), dtype=torch.float32, device="cuda:0")
    at = p if at is None else at
    at.workspace, at.workspace_size = space.data_ptr(), size
    return space, size


def run(name, p, stream=None):
    """Checks a call and runs it."""
    _, lib = R.binding()
    error = lib.op(name, "get_error")(ctypes.byref(p))
    assert error is None, error
    if stream is None:
        lib.op(name, "run")(ctypes.byref(p))
    else:
        lib.op(name, "run_async")(ctypes.byref(p), stream)
