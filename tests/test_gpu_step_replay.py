"""A whole step with drafted tokens (plan, append with norm, attention of trees, kept rows) captured once and replayed as
lengths, trees and accepted paths change. Its lengths go round in two arrays: the plan reads kv_len and writes with_new,
append, attention and keep read with_new, and keep writes kv_len, which the next step's plan reads."""

import ctypes
import math

import numpy as np
import pytest

import drafted_ref as D
import paged_ref as R

pytestmark = pytest.mark.gpu
BATCH, NODES, PAGE, HEADS, KV_HEADS, DIM, MOST = 6, 7, 8, 4, 2, 64, 160
N = HEADS + 2 * KV_HEADS
ROWS = BATCH * NODES


class Step:
    """The buffers of a step and its four calls."""

    def __init__(self, cache, pages):
        import torch

        mod, lib = R.binding()
        self.lib, self.cache, self.pages = lib, cache, pages
        ints = lambda *n: torch.zeros(n, dtype=torch.int32, device="cuda:0")  # noqa: E731
        self.per = MOST // PAGE
        self.new_len, self.parent, self.paths, self.path_len = ints(BATCH), ints(ROWS), ints(BATCH, NODES), ints(BATCH)
        self.kv_len, self.with_new, self.held, self.refused = ints(BATCH), ints(BATCH), ints(BATCH), ints(1)
        self.table = ints(BATCH, self.per) - 1
        order = np.random.default_rng(1).permutation(pages).astype(np.int32)
        self.free, self.count = R.dev(order), ints(1) + pages
        self.q_start, self.positions, self.mask = ints(BATCH + 1), ints(ROWS), ints(ROWS, 1)
        self.slots = torch.zeros(ROWS, dtype=torch.int64, device="cuda:0")
        dt = torch.int8 if cache == "qsi8dx" else torch.float16
        self.k, self.v = (torch.zeros((pages, PAGE, KV_HEADS, DIM), dtype=dt, device="cuda:0") for _ in range(2))
        self.sk = self.sv = None
        if cache == "qsi8dx":
            self.sk, self.sv = (torch.zeros((pages, KV_HEADS, PAGE), device="cuda:0") for _ in range(2))
        self.rope = R.dev(R.rope_table(MOST, DIM).astype(np.float32))
        self.w = [R.dev((1 + 0.2 * np.random.default_rng(i).standard_normal(DIM)).astype(np.float32)) for i in (2, 3)]
        self.qkv = torch.zeros((ROWS, N, DIM), dtype=torch.float16, device="cuda:0")
        self.q, self.out = (torch.zeros((ROWS, HEADS, DIM), dtype=torch.float16, device="cuda:0") for _ in range(2))
        plan = mod.PagedPlanParams(
            batch=BATCH, tokens=ROWS, page_size=PAGE, num_pages=pages, new_len=R.ptr(self.new_len),
            kv_len=R.ptr(self.kv_len), kv_len_out=R.ptr(self.with_new), held=R.ptr(self.held), held_out=R.ptr(self.held),
            block_table=R.ptr(self.table), ld_table=self.per, free_pages=R.ptr(self.free), free_capacity=pages,
            free_count=R.ptr(self.count), free_count_out=R.ptr(self.count), refused=R.ptr(self.refused),
            q_start=R.ptr(self.q_start), positions=R.ptr(self.positions), slots=R.ptr(self.slots),
            parent=R.ptr(self.parent), mask=R.ptr(self.mask), ld_mask=1)
        self.space = [D.workspace(lib, "paged_plan", plan)[0]]
        append = self.append(self.qkv, self.positions, self.slots, self.q, self.k, self.v, self.sk, self.sv)
        tree = mod.AttnTreeParams(
            attn=mod.AttnPagedParams(
                batch=BATCH, q_tokens=ROWS, q_heads=HEADS, max_q_len=NODES, max_kv_len=MOST, Q=R.ptr(self.q),
                q_token_stride=HEADS * DIM, q_head_stride=DIM, D=R.ptr(self.out), d_token_stride=HEADS * DIM,
                d_head_stride=DIM, q_start=R.ptr(self.q_start), kv_len=R.ptr(self.with_new),
                block_table=R.ptr(self.table), ld_table=self.per, scale=1.0 / math.sqrt(DIM), causal=1,
                kv=R.paged(mod, self.k, self.v, self.sk, self.sv)),
            mask=R.ptr(self.mask), ld_mask=1)
        self.space.append(D.workspace(lib, "attn_tree", tree, tree.attn)[0])
        keep = mod.KVKeepParams(
            batch=BATCH, max_keep=NODES, q_start=R.ptr(self.q_start), kv_len=R.ptr(self.with_new),
            kv_len_out=R.ptr(self.kv_len), keep=R.ptr(self.paths), ld_keep=NODES, keep_len=R.ptr(self.path_len),
            block_table=R.ptr(self.table), ld_table=self.per, layers=1, positions=R.ptr(self.positions), tokens=ROWS,
            kv=R.paged(mod, self.k, self.v, self.sk, self.sv))
        kind = "qsi8dx" if cache == "qsi8dx" else "f16"
        self.calls = [("paged_plan", plan), ("kv_append_norm_rope_%s_f16" % kind, append),
                      ("attn_tree_f16_" + kind, tree), ("kv_keep_" + kind, keep)]

    def append(self, qkv, positions, slots, q, k, v, sk, sv):
        mod, _ = R.binding()
        at = lambda h: qkv.data_ptr() + h * DIM * 2  # noqa: E731
        strides = dict(k_token_stride=N * DIM, k_head_stride=DIM, v_token_stride=N * DIM, v_head_stride=DIM,
                       q_token_stride=N * DIM, q_head_stride=DIM, qo_token_stride=HEADS * DIM, qo_head_stride=DIM)
        return mod.KVAppendNormRopeParams(
            append=mod.KVAppendRopeParams(
                tokens=qkv.shape[0], K=at(HEADS), V=at(HEADS + KV_HEADS), q_heads=HEADS, Q=at(0), Q_out=R.ptr(q),
                positions=R.ptr(positions), slots=R.ptr(slots), map=R.rope_map(mod, self.rope, DIM, False),
                kv=R.paged(mod, k, v, sk, sv), **strides),
            q_norm=D.head_norm(mod, self.w[0], 0.0, 1e-6), k_norm=D.head_norm(mod, self.w[1], 0.0, 1e-6))

    def run(self, stream):
        for name, p in self.calls:
            D.run(name, p, stream)

    def rows(self, b, n):
        """The first n tokens of sequence b in the cache, and their scales."""
        import torch

        slot = (self.table[b].long()[:, None] * PAGE + torch.arange(PAGE, device="cuda:0")).flatten()[:n]
        got = [x.flatten(0, 1)[slot] for x in (self.k, self.v)]
        return got + [x.transpose(1, 2).flatten(0, 1)[slot] for x in (self.sk, self.sv) if x is not None]

    def history(self, qkv):
        """What the cache of a sequence has to hold that was appended token by token, without drafted ones."""
        import torch

        n = qkv.shape[0]
        pos = torch.arange(n, dtype=torch.int32, device="cuda:0")
        pages = -(-n // PAGE)
        k, v = (torch.zeros((pages, PAGE, KV_HEADS, DIM), dtype=self.k.dtype, device="cuda:0") for _ in range(2))
        sk = sv = None
        if self.sk is not None:
            sk, sv = (torch.zeros((pages, KV_HEADS, PAGE), device="cuda:0") for _ in range(2))
        q = torch.empty((n, HEADS, DIM), dtype=torch.float16, device="cuda:0")
        D.run(self.calls[1][0], self.append(qkv, pos, pos.long(), q, k, v, sk, sv))
        return [x.flatten(0, 1)[:n] for x in (k, v)] + [
            x.transpose(1, 2).flatten(0, 1)[:n] for x in (sk, sv) if x is not None]


@pytest.mark.parametrize("cache", ["f16", "qsi8dx"])
@pytest.mark.parametrize("pages", [BATCH * MOST // PAGE, 17])
def test_replayed_steps_keep_what_was_accepted(gpu, cache, pages):
    """Partly accepted trees, sequences that end and begin again, and with 17 pages ones that are refused."""
    import torch

    graphed, eager = Step(cache, pages), Step(cache, pages)
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        graphed.run(torch.cuda.current_stream().cuda_stream)
    rng = np.random.default_rng(pages)
    lens, history, refusals, ends = [0] * BATCH, [None] * BATCH, 0, 0
    for step in range(24):
        new = [-1 if lens[b] > 100 or (lens[b] and rng.random() < 0.07) else int(rng.integers(0, NODES + 1))
               for b in range(BATCH)]
        count = [max(n, 0) for n in new]
        starts = np.concatenate(([0], np.cumsum(count)))
        parents = [D.random_parents(rng, n, 0.5) for n in count]
        paths = [D.path(p, int(rng.integers(0, n)))[::-1] if n else [] for p, n in zip(parents, count)]
        lists = np.full((BATCH, NODES), -1, np.int32)
        for b, x in enumerate(paths):
            lists[b, :len(x)] = x
        qkv = torch.randn((ROWS, N, DIM), device="cuda:0").half()
        parent = np.full(ROWS, -1, np.int32)
        parent[:starts[-1]] = np.concatenate(parents)
        want = D.plan(np.array(new), np.array(lens), *(R.host(x).astype(np.int64) for x in (
            graphed.held, graphed.table, graphed.free)), int(graphed.count), ROWS, PAGE, pages, parent, 1)
        for s in (graphed, eager):
            for x, y in ((s.new_len, np.array(new, np.int32)), (s.parent, parent), (s.paths, lists),
                         (s.path_len, np.array([len(x) for x in paths], np.int32))):
                x.copy_(R.dev(y))
            s.qkv.copy_(qkv)
            s.out.fill_(9.0)
            for space in s.space:
                space.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        eager.run(torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        for b in range(BATCH):
            if new[b] < 0:
                lens[b], history[b] = 0, None
                ends += 1
            elif want["kv_len_out"][b] == lens[b] + count[b]:
                x = qkv[[int(starts[b]) + i for i in paths[b]]]
                history[b] = x if history[b] is None else torch.cat((history[b], x))
                lens[b] += len(paths[b])
        refusals += int(want["refused"][0])
        for s in (graphed, eager):
            assert s.kv_len.tolist() == lens, step
            assert s.with_new.tolist() == want["kv_len_out"].tolist()
            assert s.held.tolist() == want["held_out"].tolist() and s.count.tolist() == want["free_count_out"].tolist()
            assert int(s.refused) == want["refused"][0]
            np.testing.assert_array_equal(R.host(s.table), want["table"])
        assert torch.equal(graphed.out, eager.out) and torch.isfinite(graphed.out).all()
        assert (graphed.out[int(starts[-1]):] == 9).all()
        for b in range(BATCH):
            if lens[b]:
                assert len(history[b]) == lens[b]
                for got, exact in zip(graphed.rows(b, lens[b]), graphed.history(history[b].contiguous())):
                    assert torch.equal(got, exact), (step, b)
    assert ends >= 3 and (refusals > 5) == (pages == 17)
