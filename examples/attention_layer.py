"""One attention layer of a quantized transformer on the library: a prompt prefilled in chunks, then tokens decoded one
by one, for a small batch of sequences. (With --int8-cache torch casts the QKV product's f32 rows to the f16 that the
append to an int8 cache takes.)

    python examples/attention_layer.py [--int8-cache] [--tokens N]

Each step is four calls on one stream:
  QKV product      W4A16, f32 results        (tqt_run_gemm_1xnbias_clamp_f32_f16_qsi4c2t)
  append           rotates K and Q, fills the paged cache           (tqt_run_kv_append_rope_*)
  attention        over the cache            (tqt_run_attn_paged_*)
  output product   W4A16
and at the end the decoded rows are compared with the same layer in plain torch (64-bit) from the whole
history. Weights and inputs are random.
"""

import argparse
import ctypes
import importlib.util
import math
import os

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADS, KV_HEADS, DIM, HIDDEN, BLOCK = 8, 2, 64, 512, 32
PAGE, MAX_LEN = 16, 512


def binding():
    spec = importlib.util.spec_from_file_location(
        "tqt_gfx950", os.path.join(ROOT, "torq-tile_amd", "tqt_gfx950.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod, mod.load()


class Linear:
    """int4 weights [n, k] with an f16 scale for every 32 of them."""

    def __init__(self, lib, n, k, g):
        self.run = lib.fn("w4a16f", "run_async")
        self.n, self.k = n, k
        self.q = torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
        self.s = (torch.rand((n, k // BLOCK), generator=g, device="cuda") * 0.01 + 0.002).half()
        self.bias = torch.zeros(n, device="cuda")

    def __call__(self, x, y, stream):
        m = x.shape[0]
        self.run(m, self.n, self.k, BLOCK, x.data_ptr(), self.k, 0, self.q.data_ptr(), self.k, 0,
                 self.s.data_ptr(), self.k // BLOCK, None, self.n, y.data_ptr(), self.n,
                 self.bias.data_ptr(), -math.inf, math.inf, stream)

    def exact(self, x):
        w = torch.stack((self.q & 15, self.q >> 4), 2).reshape(self.n, self.k).double() - 8
        return x.double() @ (w * self.s.double().repeat_interleave(BLOCK, 1)).T


class Layer:
    def __init__(self, batch, int8_cache):
        self.mod, self.lib = binding()
        mod = self.mod
        g = torch.Generator(device="cuda").manual_seed(1)
        self.qkv = Linear(self.lib, (HEADS + 2 * KV_HEADS) * DIM, HIDDEN, g)
        self.out = Linear(self.lib, HIDDEN, HEADS * DIM, g)
        # the table of positions, with contexts four times the model's own by interpolation
        self.table = torch.empty((MAX_LEN, DIM), device="cuda")
        t = mod.RopeTableParams(table=self.table.data_ptr(), max_pos=MAX_LEN, rotary_dim=DIM,
                                scaling=mod.ROPE_LINEAR, base=10000.0, factor=4.0)
        self.lib.op("rope_table_f32", "run")(ctypes.byref(t))
        # the cache: pages for every sequence, in a shuffled order
        per = MAX_LEN // PAGE
        pages = batch * per
        cache = torch.int8 if int8_cache else torch.float16
        self.k, self.v = (torch.zeros((pages, PAGE, KV_HEADS, DIM), dtype=cache, device="cuda")
                          for _ in range(2))
        self.sk = self.sv = None
        if int8_cache:
            self.sk, self.sv = (torch.zeros((pages, KV_HEADS, PAGE), device="cuda") for _ in range(2))
        self.pages = torch.randperm(pages, generator=g, device="cuda").to(torch.int32).view(batch, per)
        self.kv = mod.PagedKV(
            k=self.k.data_ptr(), v=self.v.data_ptr(),
            scale_k=self.sk.data_ptr() if int8_cache else None,
            scale_v=self.sv.data_ptr() if int8_cache else None, num_pages=pages, page_size=PAGE,
            kv_heads=KV_HEADS, head_dim=DIM, page_stride=self.k.stride(0), token_stride=self.k.stride(1),
            head_stride=self.k.stride(2))
        # an int8 cache takes f16 rows, an f16 one the product's f32 results as they are
        self.append = self.lib.op("kv_append_rope_" + ("qsi8dx_f16" if int8_cache else "f16_f32"), "run_async")
        self.attend = self.lib.op("attn_paged_f16_" + ("qsi8dx" if int8_cache else "f16"), "run_async")
        self.int8_cache = int8_cache

    def step(self, x, new, lengths):
        """x [tokens, HIDDEN] f16: `new[b]` tokens of every sequence, which then has lengths[b]."""
        mod, stream = self.mod, torch.cuda.current_stream().cuda_stream
        tokens, n = x.shape[0], HEADS + 2 * KV_HEADS
        seq = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new))
        pos = torch.cat([torch.arange(l - q, l) for q, l in zip(new, lengths)])
        pages = self.pages.cpu()
        slots = (pages[seq, pos // PAGE].long() * PAGE + pos % PAGE).cuda()
        pos = pos.to(torch.int32).cuda()
        start = torch.tensor([0] + new).cumsum(0).to(torch.int32).cuda()
        kv_len = torch.tensor(lengths, dtype=torch.int32).cuda()

        qkv = torch.empty((tokens, n, DIM), device="cuda")
        self.qkv(x, qkv, stream)
        rows = qkv.half() if self.int8_cache else qkv
        q = torch.empty((tokens, HEADS, DIM), dtype=torch.float16, device="cuda")
        at = lambda head: rows.data_ptr() + head * DIM * rows.element_size()  # noqa: E731
        a = mod.KVAppendRopeParams(
            tokens=tokens, K=at(HEADS), k_token_stride=n * DIM, k_head_stride=DIM,
            V=at(HEADS + KV_HEADS), v_token_stride=n * DIM, v_head_stride=DIM, q_heads=HEADS, Q=at(0),
            q_token_stride=n * DIM, q_head_stride=DIM, Q_out=q.data_ptr(), qo_token_stride=HEADS * DIM,
            qo_head_stride=DIM, positions=pos.data_ptr(), slots=slots.data_ptr(),
            map=mod.RopeMap(table=self.table.data_ptr(), max_pos=MAX_LEN, rotary_dim=DIM), kv=self.kv)
        self.append(ctypes.byref(a), stream)

        o = torch.empty((tokens, HEADS * DIM), dtype=torch.float16, device="cuda")
        p = mod.AttnPagedParams(
            batch=len(new), q_tokens=tokens, q_heads=HEADS, max_q_len=max(new), max_kv_len=max(lengths),
            Q=q.data_ptr(), q_token_stride=HEADS * DIM, q_head_stride=DIM, D=o.data_ptr(),
            d_token_stride=HEADS * DIM, d_head_stride=DIM, q_start=start.data_ptr(),
            kv_len=kv_len.data_ptr(), block_table=self.pages.data_ptr(), ld_table=self.pages.stride(0),
            scale=1.0 / math.sqrt(DIM), causal=1, kv=self.kv)
        size = self.lib.op("attn_paged", "get_workspace_size")(ctypes.byref(p))
        space = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
        p.workspace, p.workspace_size = space.data_ptr(), size
        self.attend(ctypes.byref(p), stream)

        y = torch.empty((tokens, HIDDEN), device="cuda")
        self.out(o, y, stream)
        return y

    def exact(self, x):
        """The layer over one sequence's whole history x [tokens, HIDDEN], in 64 bits."""
        n = x.shape[0]
        qkv = self.qkv.exact(x).view(n, -1, DIM)
        c, s = self.table[:n, :DIM // 2].double()[:, None], self.table[:n, DIM // 2:].double()[:, None]
        a, b = qkv[:, :HEADS + KV_HEADS, :DIM // 2], qkv[:, :HEADS + KV_HEADS, DIM // 2:]
        qk = torch.cat((a * c - b * s, b * c + a * s), -1)
        q, k, v = qk[:, :HEADS], qk[:, HEADS:], qkv[:, HEADS + KV_HEADS:]
        k, v = (t.repeat_interleave(HEADS // KV_HEADS, 1) for t in (k, v))
        w = torch.einsum("ihd,jhd->hij", q, k) / math.sqrt(DIM)
        w = w.masked_fill(torch.ones((n, n), device="cuda").triu(1).bool(), -math.inf).softmax(-1)
        return self.out.exact(torch.einsum("hij,jhd->ihd", w, v).reshape(n, -1))


def run(int8_cache=False, decode=8, prompts=(70, 5, 130), chunk=48):
    """Relative error of the last decoded rows against the exact layer."""
    layer = Layer(len(prompts), int8_cache)
    g = torch.Generator(device="cuda").manual_seed(2)
    history = [torch.randn((p + decode, HIDDEN), generator=g, device="cuda").half() for p in prompts]
    done = [0] * len(prompts)
    # chunks of the prompts, short ones decoding beside long ones; then a token each
    while min(d - p for d, p in zip(done, prompts)) < decode:
        new = [min(chunk, p - d) if d < p else int(d < p + decode) for d, p in zip(done, prompts)]
        x = torch.cat([h[d:d + q] for h, d, q in zip(history, done, new)])
        done = [d + q for d, q in zip(done, new)]
        y = layer.step(x, new, done)
        ends = torch.tensor(new).cumsum(0) - 1
        for b, q in enumerate(new):
            if q > 0 and done[b] == prompts[b] + decode:
                last = y[ends[b]].double()
                want = layer.exact(history[b])[-1]
                yield b, done[b], float((last - want).norm() / want.norm())


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--int8-cache", action="store_true")
    ap.add_argument("--tokens", type=int, default=8)
    args = ap.parse_args()
    for b, n, err in run(args.int8_cache, args.tokens):
        print("sequence %d, %d tokens: relative error %.2e" % (b, n, err), flush=True)
