"""One attention layer decoding with drafted tokens on the library: prompts, then steps in which every sequence
brings a tree of drafted tokens, some path of it is accepted, and the cache keeps that path's rows. Heads of Q and K
are normalised. (Which path is accepted is drawn at random here; a model's own choice would stand there.)

    python examples/drafted_layer.py [--int8-cache] [--steps N]

Each step is six calls on one stream, and nothing of it comes back to the host:
  plan             pages, block table, slots, positions, tree masks  (tqt_run_paged_plan)
  QKV product      W4A16, f32 results                        (tqt_run_gemm_1xnbias_clamp_f32_f16_qsi4c2t)
  append           norm and rotation of K and Q, fills the paged cache  (tqt_run_kv_append_norm_rope_*)
  attention        of the trees over the cache               (tqt_run_attn_tree_*; prompts: tqt_run_attn_paged_*)
  output product   W4A16
  keep             the accepted rows of the cache            (tqt_run_kv_keep_*)
and at the end the accepted rows' outputs are compared with the same layer in plain torch (64-bit) over the
accepted history. Weights and inputs are random.
"""

import argparse
import ctypes
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from attention_layer import DIM, HEADS, HIDDEN, KV_HEADS, MAX_LEN, PAGE, Linear, binding  # noqa: E402

EPS, NODES = 1e-6, 12


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class Layer:
    def __init__(self, batch, int8_cache):
        self.mod, self.lib = binding()
        mod = self.mod
        g = torch.Generator(device="cuda").manual_seed(1)
        self.qkv = Linear(self.lib, (HEADS + 2 * KV_HEADS) * DIM, HIDDEN, g)
        self.out = Linear(self.lib, HIDDEN, HEADS * DIM, g)
        self.wq, self.wk = (1 + 0.2 * torch.randn(DIM, generator=g, device="cuda") for _ in range(2))
        self.table = torch.empty((MAX_LEN, DIM), device="cuda")
        t = mod.RopeTableParams(table=self.table.data_ptr(), max_pos=MAX_LEN, rotary_dim=DIM, base=10000.0)
        self.lib.op("rope_table_f32", "run")(ctypes.byref(t))
        # the cache, all of its pages free at first
        self.per = MAX_LEN // PAGE
        self.num_pages = batch * self.per
        cache = torch.int8 if int8_cache else torch.float16
        self.k, self.v = (torch.zeros((self.num_pages, PAGE, KV_HEADS, DIM), dtype=cache, device="cuda")
                          for _ in range(2))
        self.sk = self.sv = None
        if int8_cache:
            self.sk, self.sv = (torch.zeros((self.num_pages, KV_HEADS, PAGE), device="cuda") for _ in range(2))
        self.kv = mod.PagedKV(
            k=self.k.data_ptr(), v=self.v.data_ptr(), scale_k=self.sk.data_ptr() if int8_cache else None,
            scale_v=self.sv.data_ptr() if int8_cache else None, num_pages=self.num_pages, page_size=PAGE,
            kv_heads=KV_HEADS, head_dim=DIM, page_stride=self.k.stride(0), token_stride=self.k.stride(1),
            head_stride=self.k.stride(2))
        self.free = torch.randperm(self.num_pages, generator=g, device="cuda").to(torch.int32)
        self.free_count = ints([self.num_pages])
        self.blocks = torch.full((batch, self.per), -1, dtype=torch.int32, device="cuda")
        self.held, self.refused = ints([0] * batch), ints([0])
        self.kv_len, self.with_drafted = ints([0] * batch), ints([0] * batch)
        self.int8_cache, self.batch = int8_cache, batch

    def op(self, name, p, stream):
        self.lib.op(name, "run_async")(ctypes.byref(p), stream)

    def space(self, name, p, at):
        """The call's workspace (a program would keep one of the largest size)."""
        size = self.lib.op(name, "get_workspace_size")(ctypes.byref(p))
        space = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
        at.workspace, at.workspace_size = space.data_ptr(), size
        return space

    def step(self, x, new, most_keys, parent=None):
        """x [tokens, HIDDEN] f16, new[b] tokens of every sequence (-1: it has ended); parent: their trees."""
        mod, stream = self.mod, torch.cuda.current_stream().cuda_stream
        tokens, most = x.shape[0], max(max(new), 1)
        new_len, self.q_start = ints(new), torch.empty(self.batch + 1, dtype=torch.int32, device="cuda")
        positions = self.positions = torch.empty(tokens, dtype=torch.int32, device="cuda")
        slots = torch.empty(tokens, dtype=torch.int64, device="cuda")
        mask = torch.empty((tokens, 1), dtype=torch.int32, device="cuda")
        p = mod.PagedPlanParams(
            batch=self.batch, tokens=tokens, page_size=PAGE, num_pages=self.num_pages, new_len=new_len.data_ptr(),
            kv_len=self.kv_len.data_ptr(), kv_len_out=self.with_drafted.data_ptr(), held=self.held.data_ptr(),
            held_out=self.held.data_ptr(), block_table=self.blocks.data_ptr(), ld_table=self.per,
            free_pages=self.free.data_ptr(), free_capacity=self.num_pages, free_count=self.free_count.data_ptr(),
            free_count_out=self.free_count.data_ptr(), refused=self.refused.data_ptr(),
            q_start=self.q_start.data_ptr(), positions=positions.data_ptr(), slots=slots.data_ptr())
        if parent is not None:
            p.parent, p.mask, p.ld_mask = parent.data_ptr(), mask.data_ptr(), 1
        keep = [self.space("paged_plan", p, p)]
        self.op("paged_plan", p, stream)

        n = HEADS + 2 * KV_HEADS
        qkv = torch.empty((tokens, n, DIM), device="cuda")
        self.qkv(x, qkv, stream)
        rows = qkv.half() if self.int8_cache else qkv
        q = torch.empty((tokens, HEADS, DIM), dtype=torch.float16, device="cuda")
        at = lambda head: rows.data_ptr() + head * DIM * rows.element_size()  # noqa: E731
        a = mod.KVAppendNormRopeParams(
            append=mod.KVAppendRopeParams(
                tokens=tokens, K=at(HEADS), k_token_stride=n * DIM, k_head_stride=DIM, V=at(HEADS + KV_HEADS),
                v_token_stride=n * DIM, v_head_stride=DIM, q_heads=HEADS, Q=at(0), q_token_stride=n * DIM,
                q_head_stride=DIM, Q_out=q.data_ptr(), qo_token_stride=HEADS * DIM, qo_head_stride=DIM,
                positions=positions.data_ptr(), slots=slots.data_ptr(),
                map=mod.RopeMap(table=self.table.data_ptr(), max_pos=MAX_LEN, rotary_dim=DIM), kv=self.kv),
            q_norm=mod.HeadNorm(weight=self.wq.data_ptr(), eps=EPS),
            k_norm=mod.HeadNorm(weight=self.wk.data_ptr(), eps=EPS))
        self.op("kv_append_norm_rope_" + ("qsi8dx_f16" if self.int8_cache else "f16_f32"), a, stream)

        o = torch.empty((tokens, HEADS * DIM), dtype=torch.float16, device="cuda")
        t = mod.AttnPagedParams(
            batch=self.batch, q_tokens=tokens, q_heads=HEADS, max_q_len=most, max_kv_len=most_keys, Q=q.data_ptr(),
            q_token_stride=HEADS * DIM, q_head_stride=DIM, D=o.data_ptr(), d_token_stride=HEADS * DIM,
            d_head_stride=DIM, q_start=self.q_start.data_ptr(), kv_len=self.with_drafted.data_ptr(),
            block_table=self.blocks.data_ptr(), ld_table=self.per, scale=1.0 / math.sqrt(DIM), causal=1, kv=self.kv)
        cache = "f16_" + ("qsi8dx" if self.int8_cache else "f16")
        if parent is None:
            keep.append(self.space("attn_paged", t, t))
            self.op("attn_paged_" + cache, t, stream)
        else:
            tree = mod.AttnTreeParams(attn=t, mask=mask.data_ptr(), ld_mask=1)
            keep.append(self.space("attn_tree", tree, tree.attn))
            self.op("attn_tree_" + cache, tree, stream)
        y = torch.empty((tokens, HIDDEN), device="cuda")
        self.out(o, y, stream)
        return y

    def keep(self, path, path_len):
        """path [batch, n]: the accepted tokens' numbers, path_len of them."""
        c = self.mod.KVKeepParams(
            batch=self.batch, max_keep=path.shape[1], q_start=self.q_start.data_ptr(),
            kv_len=self.with_drafted.data_ptr(), kv_len_out=self.kv_len.data_ptr(), keep=path.data_ptr(),
            ld_keep=path.stride(0), keep_len=path_len.data_ptr(), block_table=self.blocks.data_ptr(),
            ld_table=self.per, layers=1, kv=self.kv, positions=self.positions.data_ptr(),
            tokens=self.positions.numel())
        self.op("kv_keep_" + ("qsi8dx" if self.int8_cache else "f16"), c, torch.cuda.current_stream().cuda_stream)

    def exact(self, x):
        """The layer over one sequence's accepted history x [tokens, HIDDEN], in 64 bits."""
        n = x.shape[0]
        qkv = self.qkv.exact(x).view(n, -1, DIM)

        def head(h, w):
            h = h / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS) * w.double()
            c, s = (self.table[:n, i:i + DIM // 2].double()[:, None] for i in (0, DIM // 2))
            a, b = h[..., :DIM // 2], h[..., DIM // 2:]
            return torch.cat((a * c - b * s, b * c + a * s), -1)

        q, k = head(qkv[:, :HEADS], self.wq), head(qkv[:, HEADS:HEADS + KV_HEADS], self.wk)
        k, v = (t.repeat_interleave(HEADS // KV_HEADS, 1) for t in (k, qkv[:, HEADS + KV_HEADS:]))
        w = torch.einsum("ihd,jhd->hij", q, k) / math.sqrt(DIM)
        w = w.masked_fill(torch.ones((n, n), device="cuda").triu(1).bool(), -math.inf).softmax(-1)
        return self.out.exact(torch.einsum("hij,jhd->ihd", w, v).reshape(n, -1))


def run(int8_cache=False, steps=6, prompts=(70, 5, 130)):
    """Every accepted row's relative error against the exact layer; the second sequence ends halfway, and another one
    with a prompt of its own takes its place and its pages."""
    batch = len(prompts)
    layer = Layer(batch, int8_cache)
    g = torch.Generator(device="cuda").manual_seed(2)
    draw = torch.Generator().manual_seed(3)
    hidden = lambda n: torch.randn((n, HIDDEN), generator=g, device="cuda").half()  # noqa: E731
    number = lambda lo, hi: int(torch.randint(lo, hi + 1, (1,), generator=draw))  # noqa: E731

    def prompt(lengths):
        x = [hidden(max(n, 0)) for n in lengths]
        layer.step(torch.cat(x), lengths, MAX_LEN)
        layer.kv_len.copy_(layer.with_drafted)
        return x

    history, checks = prompt(list(prompts)), []
    for step in range(steps):
        if step == steps // 2:
            layer.step(hidden(1), [1 if b == 0 else -1 if b == 1 else 0 for b in range(batch)], MAX_LEN)
            layer.kv_len[1:2].copy_(layer.with_drafted[1:2])  # the token beside it is not kept
            history[1] = prompt([37 if b == 1 else 0 for b in range(batch)])[1]
        new = [number(2, NODES) for _ in range(batch)]
        parents = [[-1] + [number(0, i - 1) for i in range(1, n)] for n in new]
        x = [hidden(n) for n in new]
        y = layer.step(torch.cat(x), new, MAX_LEN, ints(sum(parents, [])))
        paths = []
        for b, n in enumerate(new):
            path = [number(0, n - 1)]
            while parents[b][path[0]] >= 0:
                path.insert(0, parents[b][path[0]])
            paths.append(path)
        most = max(len(p) for p in paths)
        layer.keep(ints([p + [0] * (most - len(p)) for p in paths]), ints([len(p) for p in paths]))
        for b, row in enumerate(torch.tensor([0] + new).cumsum(0)[:-1].tolist()):
            history[b] = torch.cat((history[b], x[b][paths[b]]))
            checks.append((step, b, history[b], y[row + paths[b][-1]].double()))
    assert int(layer.refused) == 0
    assert layer.kv_len.tolist() == [h.shape[0] for h in history]
    for step, b, h, row in checks:
        want = layer.exact(h)[-1]
        yield step, b, h.shape[0], float((row - want).norm() / want.norm())


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--int8-cache", action="store_true")
    ap.add_argument("--steps", type=int, default=6)
    args = ap.parse_args()
    for step, b, n, err in run(args.int8_cache, args.steps):
        print("step %d, sequence %d, %d tokens: relative error %.2e" % (step, b, n, err), flush=True)
