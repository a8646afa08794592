"""Plain 64-bit forms of the rotary, cache-append and attention operators, and builders of their calls
(test infrastructure). Numpy only; the builders take torch tensors on the GPU."""

import ctypes
import functools
import math

import numpy as np

import tqt_testlib as T

# unit roundoff and the spacing below the smallest normal number
ROUND = {"f32": (2.0 ** -24, 2.0 ** -149), "f16": (2.0 ** -11, 2.0 ** -24),
         "bf16": (2.0 ** -8, 2.0 ** -133)}


@functools.lru_cache(maxsize=None)
def binding():
    mod = T.load_product_module()
    return mod, mod.load()


def rope_table(max_pos, rot, base=10000.0, freq=None):
    """[max_pos, rot] f64: cosines, then sines."""
    half = rot // 2
    f = base ** (-2.0 * np.arange(half) / rot) if freq is None else freq
    a = np.arange(max_pos, dtype=np.float64)[:, None] * f
    return np.concatenate((np.cos(a), np.sin(a)), 1)


def pairs(rot, interleaved):
    """Element indexes (first, second) of every pair."""
    i = np.arange(rot // 2)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)


def rope(x, positions, table, rot, interleaved, inverse=False, dtype=np.float64):
    """x [tokens, heads, d] and the size of the terms of every result (for its rounding bound). With
    dtype float32 every product and sum is rounded on its own, as the library defines it."""
    y = x.astype(dtype).copy()
    size = np.abs(y)
    if rot:
        t = table.astype(dtype)[positions]
        c, s = t[:, None, :rot // 2], t[:, None, rot // 2:]
        if inverse:
            s = -s
        e1, e2 = pairs(rot, interleaved)
        a, b = y[..., e1].copy(), y[..., e2].copy()
        y[..., e1] = a * c - b * s
        y[..., e2] = b * c + a * s
        size[..., e1] = np.abs(a * c) + np.abs(b * s)
        size[..., e2] = np.abs(b * c) + np.abs(a * s)
    return y, size


def quantize_rows(rows):
    """Symmetric int8 of f32 rows [..., d], as the library defines it: (q, scale)."""
    amax = np.abs(rows).max(-1)
    scale = (amax * (np.float32(1) / np.float32(127))).astype(np.float32)
    zero = scale == 0
    scale = np.where(zero, np.float32(1), scale)
    with np.errstate(over="ignore"):
        q = np.clip(np.rint(rows / scale[..., None]), -127, 127)
    q[zero] = 0
    return q.astype(np.int8), scale


def visible(nq, nk, causal, window):
    """[nq, nk]: which keys each query sees by position."""
    pos = nk - nq + np.arange(nq)[:, None]
    j = np.arange(nk)[None]
    see = np.ones((nq, nk), bool)
    if causal:
        see &= j <= pos
    if window:
        see &= j > pos - window
    return see


def attention(q, k, v, see, scale):
    """q [nq, h, d], k / v [nk, kh, d] f64, see [nq, nk] -> out, lse, and what bounds their error: the
    weighted |v|, the largest |v| seen over the sum, the size of the terms of a score."""
    nq, h, d = q.shape
    kh = k.shape[1]
    out = np.zeros((nq, h, d))
    lse = np.full((nq, h), -np.inf)
    weight, top, terms = np.zeros((nq, h, d)), np.zeros((nq, h, d)), np.zeros((nq, h))
    for i in range(nq):
        keys = np.nonzero(see[i])[0]
        if len(keys) == 0:
            continue
        for hh in range(h):
            kk, vv = k[keys, hh // (h // kh)], v[keys, hh // (h // kh)]
            s = (kk @ q[i, hh]) * scale
            terms[i, hh] = np.max(np.abs(kk) @ np.abs(q[i, hh])) * abs(scale)
            m = s.max()
            if m == -np.inf:
                continue
            p = np.exp(s - m)
            out[i, hh] = p @ vv / p.sum()
            weight[i, hh] = p @ np.abs(vv) / p.sum()
            top[i, hh] = np.abs(vv).max(0) * len(keys) / p.sum()
            lse[i, hh] = m + math.log(p.sum())
    return out, lse, weight, top, terms


def attention_bound(kind, d, out, lse, weight, top, terms):
    """How far D and lse may be from 64 bits. A score is a sum of d exact products in f32: its terms times
    d 2^-24, and a few roundings of scale and exp. A probability is rounded to the type (and, below its
    normal range, by half its smallest step), the result once more."""
    u, tiny = ROUND[kind]
    ds = terms * (d + 4) * 2.0 ** -24 + 2.0 ** -20
    ds = ds + 2.0 ** -22 * np.abs(np.where(np.isfinite(lse), lse, 0))
    tol = weight * (u + 2 * ds[..., None]) * 1.01 + u * np.abs(out) + tiny * (1 + top)
    return tol, ds * 2 + 1e-6


# ------------------------------------------------------------------------------------------
# Calls
# ------------------------------------------------------------------------------------------

def torch_type(kind):
    import torch

    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16,
            "qsi8dx": torch.int8}[kind]


def dev(a, kind=None):
    """A numpy array on the GPU, rounded to a type."""
    import torch

    t = torch.from_numpy(np.ascontiguousarray(a)).to("cuda:0")
    return t if kind is None else t.to(torch_type(kind))


def host(t):
    return t.double().cpu().numpy()


def ptr(t):
    return None if t is None else t.data_ptr()


def rope_map(mod, table, rot, interleaved, inverse=False):
    return mod.RopeMap(table=ptr(table), max_pos=0 if table is None else table.shape[0],
                       rotary_dim=rot, interleaved=int(interleaved), inverse=int(inverse))


def paged(mod, k, v, sk=None, sv=None, page=None, heads_first=False):
    """k, v [pages, page, heads, d], or [pages, heads, page, d] with heads_first."""
    tok, head = (2, 1) if heads_first else (1, 2)
    return mod.PagedKV(k=ptr(k), v=ptr(v), scale_k=ptr(sk), scale_v=ptr(sv), num_pages=k.shape[0],
                       page_size=k.shape[tok], kv_heads=k.shape[head], head_dim=k.shape[3],
                       page_stride=k.stride(0), token_stride=k.stride(tok),
                       head_stride=k.stride(head))


def run_attention(name, q, kv, q_start, kv_len, table, out, lse, scale, causal=True, window=0,
                  max_q=None, max_kv=None, stream=None, keep=None):
    """One call; q, out [tokens, heads, d] (any strides), table [batch, ld] int32. Returns the params
    (with their workspace in `keep`)."""
    import torch

    mod, lib = binding()
    starts = q_start.cpu().numpy()
    p = mod.AttnPagedParams(
        batch=len(starts) - 1, q_tokens=q.shape[0], q_heads=q.shape[1],
        max_q_len=int(np.max(starts[1:] - starts[:-1], initial=0)) if max_q is None else max_q,
        max_kv_len=int(kv_len.max()) if max_kv is None else max_kv, Q=ptr(q),
        q_token_stride=q.stride(0), q_head_stride=q.stride(1), D=ptr(out),
        d_token_stride=out.stride(0), d_head_stride=out.stride(1), lse=ptr(lse),
        q_start=ptr(q_start), kv_len=ptr(kv_len), block_table=ptr(table),
        ld_table=table.stride(0) if table.shape[0] > 1 else table.shape[1], scale=scale,
        causal=int(causal), window=window, kv=kv)
    size = lib.op("attn_paged", "get_workspace_size")(ctypes.byref(p))
    # filled with NaN: nothing may be read from it before it is written
    space = torch.full((max(size // 4, 4) + 64,), float("nan"), dtype=torch.float32, device="cuda:0")
    p.workspace, p.workspace_size = space.data_ptr(), size
    error = lib.op("attn_paged_" + name, "get_error")(ctypes.byref(p))
    assert error is None, error
    if stream is None:
        lib.op("attn_paged_" + name, "run")(ctypes.byref(p))
        assert torch.isnan(space[size // 4 + 4:]).all()  # nothing past its end is written
    else:
        lib.op("attn_paged_" + name, "run_async")(ctypes.byref(p), stream)
    if keep is not None:
        keep.append((p, space))
    return p
