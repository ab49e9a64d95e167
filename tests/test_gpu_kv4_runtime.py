"""The operators run together: prompts in chunks, decode steps, a request that leaves and one that joins, a replayed graph,
on 4-bit pools and on bf16 ones with rotary positions of several axes."""

from __future__ import annotations

from dataclasses import replace

import pytest
import torch

import attention_runtime as ar
import hip_ops
from decode_state import DeviceBatchPageTables, FullAttentionCache, SharedKV4BlockPool, SharedKVBlockPool
from oracle import kv4
from test_gpu_attention_kv4 import _attend, _close

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _config(heads, kv_heads, dim, gate=True):
    text = {"linear_num_key_heads": 1, "linear_num_value_heads": 1, "linear_key_head_dim": 4, "linear_value_head_dim": 4, "linear_conv_kernel_dim": 4,
            "num_attention_heads": heads, "num_key_value_heads": kv_heads, "head_dim": dim, "attn_output_gate": gate, "native_paged_attention": True}
    return ar.parse_attention_config({"text_config": text})


class _Layer:
    """One layer of a running batch, and what its requests have been given so far."""

    def __init__(self, seed, pool, heads, kv_heads, dim, rope):
        self.gen = torch.Generator().manual_seed(seed)
        self.pool, self.heads, self.kv_heads, self.dim, self.rope = pool, heads, kv_heads, dim, rope
        self.qw, self.kw = (self._bf(dim) * 0.3 for _ in range(2))
        self.kv = {}  # request -> keys and values (tokens, H_kv, D) before the prologue, and positions (axes, tokens)

    def _bf(self, *shape):
        return torch.randn(*shape, generator=self.gen).to(torch.bfloat16).to(DEV)

    def tokens(self, n):
        return self._bf(n, self.heads * 2 * self.dim), self._bf(n, self.kv_heads * self.dim), self._bf(n, self.kv_heads * self.dim)

    def took(self, req, k, v, positions):
        old = self.kv.get(req)
        new = (k.view(-1, self.kv_heads, self.dim), v.view(-1, self.kv_heads, self.dim), positions)
        self.kv[req] = new if old is None else (torch.cat([old[0], new[0]]), torch.cat([old[1], new[1]]), torch.cat([old[2], new[2]], 1))

    def prologue(self, q, k, v, positions):
        """The query, and the keys and values that the pool has to hold, (tokens, H_kv, D)."""
        n, block = q.shape[0], self.pool.block_size
        blocks = -(-n // block)
        tables = torch.arange(blocks, dtype=torch.int32, device=DEV).unsqueeze(0)
        kind = self.pool.key_blocks.shape[1:], self.pool.key_blocks.dtype
        pools = [torch.zeros(blocks, *kind[0], dtype=kind[1], device=DEV) for _ in range(2)]
        query, _ = hip_ops.qk_norm_mrope_kv_append(q, k, v, self.qw, self.kw, positions, self.rope.sections(self.dim), *pools, torch.arange(n, device=DEV), block,
                                                   eps=self.rope.rms_norm_eps, rope_theta=self.rope.rope_theta, interleaved=self.rope.mrope_interleaved)
        gather = hip_ops.paged_kv4_gather if kind[1] == torch.uint8 else hip_ops.paged_kv_gather
        return query, *(x[0].transpose(0, 1) for x in gather(*pools, tables, n, block))

    def check(self, req, q, out, table):
        """``out`` (n, H D): what the request's last n tokens, of projection ``q``, got; ``table``: its block ids."""
        k, v, positions = self.kv[req]
        n, total, block = q.shape[0], k.shape[0], self.pool.block_size
        all_q = torch.zeros(total, q.shape[1], dtype=torch.bfloat16, device=DEV)
        all_q[-n:] = q
        query, keys, values = self.prologue(all_q, k, v, positions)
        four = self.pool.key_blocks.dtype == torch.uint8
        got = (hip_ops.paged_kv4_gather if four else hip_ops.paged_kv_gather)(self.pool.key_blocks, self.pool.value_blocks, table.unsqueeze(0).contiguous(), total, block)
        assert torch.equal(got[0][0].transpose(0, 1), keys) and torch.equal(got[1][0].transpose(0, 1), values)
        seen = torch.arange(total, device=DEV) <= torch.arange(total - n, total, device=DEV).unsqueeze(1)
        want, mass = _attend(query[-n:].double(), keys.transpose(0, 1).double().contiguous(), values.transpose(0, 1).double().contiguous(), seen, self.dim**-0.5)
        gate = all_q[-n:].view(n, self.heads, 2 * self.dim)[..., self.dim:]
        out = out.view(n, self.heads, self.dim)
        if four:
            _close(out, want, mass, gate)
            return
        # the bf16 step rounds the heads, the sigmoid and their product, and the probabilities, each by up to 2^-8
        s = torch.sigmoid(gate.double())
        assert ((out.double() - want * s).abs() <= 2.0**-8 * (3.05 * (want * s).abs() + mass * s) + 2.0**-10 * mass * s).all()


CASES = [
    (16, 2, 256, 16, (11, 11, 10), True, "4-bit"), (20, 4, 128, 32, (16, 24, 24), False, "4-bit"), (8, 8, 128, 16, None, False, "4-bit"), (16, 2, 256, 16, (11, 11, 10), True, "bf16"),
]


@pytest.mark.parametrize("heads,kv_heads,dim,block,sections,interleaved,kind", CASES)
def test_a_running_batch(heads, kv_heads, dim, block, sections, interleaved, kind) -> None:
    rope = ar.RopeConfig(rope_theta=1e6, mrope_section=sections, mrope_interleaved=interleaved)
    config, runtime = _config(heads, kv_heads, dim), ar.HotPathRuntime()
    make = SharedKV4BlockPool if kind == "4-bit" else SharedKVBlockPool
    layers = [_Layer(seed, make(40, kv_heads, dim, block_size=block, device=DEV), heads, kv_heads, dim, rope) for seed in (1, 2)]
    tables = DeviceBatchPageTables(layers[0].pool, rows=5, max_blocks=8)
    gen = torch.Generator().manual_seed(3)
    axes = len(rope.sections(dim))
    length, row_of = {}, {}

    def spread(places):
        return torch.tensor(places, device=DEV).expand(axes, -1).contiguous()

    def chunk(counts, picture=False):
        reqs = sorted(counts, key=row_of.get)
        step = tables.plan_prefill([row_of[r] for r in reqs], [counts[r] for r in reqs])
        places = [length[r] + i for r in reqs for i in range(counts[r])]
        positions = spread(places)
        if picture:
            positions += torch.randint(-3, 9, positions.shape, generator=gen).to(DEV)
        for layer in layers:
            q, k, v = layer.tokens(len(places))
            out = ar.full_attention_prefill_device(q, k, v, layer.qw, layer.kw, layer.pool.key_blocks, layer.pool.value_blocks, step, config, runtime, rope,
                                                   positions=positions if picture else None)
            at = 0
            for r in reqs:
                part = slice(at, at + counts[r])
                at += counts[r]
                layer.took(r, k[part], v[part], positions[:, part])
                layer.check(r, q[part], out[part], tables.block_tables[row_of[r]])
        for r in reqs:
            length[r] += counts[r]

    def admit(req):
        row_of[req] = tables.add_request()
        length[req] = 0

    def decode(inputs, positions):
        plan = tables.plan_step()
        return [ar.full_attention_decode_step_device(*x, layer.qw, layer.kw, layer.pool.key_blocks, layer.pool.value_blocks, tables, config, runtime, rope, plan=plan, positions=positions)
                for layer, x in zip(layers, inputs)]

    def check_step(inputs, outs, positions):
        for layer, (q, k, v), out in zip(layers, inputs, outs):
            assert out.shape == (tables.rows, 1, heads * dim)
            for r, row in row_of.items():
                layer.took(r, k[row : row + 1], v[row : row + 1], spread([length[r]]) if positions is None else positions[:, row : row + 1])
                layer.check(r, q[row : row + 1], out[row], tables.block_tables[row])
            for row in set(range(tables.rows)) - set(row_of.values()):
                assert (out[row] == 0).all()
        for r in row_of:
            length[r] += 1

    def step(moved=False):
        positions = None
        if moved:
            at = {row: length[r] for r, row in row_of.items()}
            positions = spread([at.get(row, 0) + 5 for row in range(tables.rows)])
        inputs = [layer.tokens(tables.rows) for layer in layers]
        check_step(inputs, decode(inputs, positions), positions)

    for req in "abc":
        admit(req)
    chunk({"a": 20, "b": 5, "c": 33})
    chunk({"a": 17, "c": 37}, picture=sections is not None)
    step()
    step(moved=sections is not None)
    tables.release_request(row_of.pop("b"))
    step()
    admit("d")
    chunk({"d": 1})
    chunk({"d": 15, "a": 2})
    step()
    tables.release_request(row_of.pop("a"))  # the graph's batch has an empty row at its front
    inputs = [layer.tokens(tables.rows) for layer in layers]
    graph = torch.cuda.CUDAGraph()
    kept = [x.clone() for x in (tables.block_tables, tables.sequence_lengths, tables.allocator.free_state)]
    with torch.cuda.graph(graph):
        outs = decode(inputs, None)
    for now, before in zip((tables.block_tables, tables.sequence_lengths, tables.allocator.free_state), kept):
        assert torch.equal(now, before)
    for _ in range(3):
        for layer, x in zip(layers, inputs):
            for old, new in zip(x, layer.tokens(tables.rows)):
                old.copy_(new)
        graph.replay()
        check_step([[t.clone() for t in x] for x in inputs], outs, None)
        tables.check()
    stats = runtime.paged_attention_stats
    assert stats.native_prefill_hits == 2 * 4 and stats.native_hits == 2 * 5 and stats.dense_fallbacks == 0
    for r in list(row_of):
        tables.release_request(row_of.pop(r))
    assert tables.allocator.free_count == 40


def test_post_rotary_keys_and_values_on_a_4_bit_pool() -> None:
    heads, kv_heads, dim, block, rows = 16, 2, 256, 16, 3
    config, runtime = _config(heads, kv_heads, dim), ar.HotPathRuntime()
    pool = SharedKV4BlockPool(8, kv_heads, dim, block_size=block, device=DEV)
    tables = DeviceBatchPageTables(pool, rows=rows, max_blocks=4)
    tables.add_request()
    tables.add_request()
    gen = torch.Generator().manual_seed(4)
    seen = []
    for _ in range(3):
        bf = lambda *shape: torch.randn(*shape, generator=gen).to(torch.bfloat16).to(DEV)  # noqa: E731
        q, k, v, gate = bf(rows, heads, 1, dim), bf(rows, kv_heads, 1, dim), bf(rows, kv_heads, 1, dim), bf(rows, 1, heads * dim)
        seen.append((k, v))
        plan = tables.plan_step()
        out = ar.full_attention_decode_device(q, gate, k, v, pool.key_blocks, pool.value_blocks, tables, config, runtime, plan=plan)
        for row in (0, 1):
            keys, values = (torch.cat([torch.from_numpy(kv4.quantized(x[i][row].double().cpu().numpy())) for x in seen], 1).to(DEV) for i in (0, 1))
            want, mass = _attend(q[row].transpose(0, 1).double(), keys, values, torch.ones(1, len(seen), dtype=torch.bool, device=DEV), dim**-0.5)
            s = torch.sigmoid(gate[row].double()).view(1, heads, dim)
            # the heads, the sigmoid and the product are each rounded to bf16
            assert ((out[row].view(1, heads, dim).double() - want * s).abs() <= 2.0**-8 * (3.05 * (want * s).abs() + mass * s) + 2.0**-12 * mass * s).all()
        assert (out[2] == 0).all()


@pytest.mark.parametrize("heads,kv_heads,dim,block", [(16, 2, 256, 16), (20, 4, 128, 64)])
def test_request_caches_on_a_shared_4_bit_pool(heads, kv_heads, dim, block) -> None:
    config, runtime = _config(heads, kv_heads, dim), ar.HotPathRuntime()
    pool = SharedKV4BlockPool(24, kv_heads, dim, block_size=block, device=DEV)
    gen = torch.Generator().manual_seed(5)
    caches = [FullAttentionCache(block_size=block, shared_pool=pool) for _ in range(3)]
    dense = []
    for cache, lens in zip(caches, ((70, 1), (3, 20), (16,))):
        parts = []
        for n in lens:
            k, v = (torch.randn(1, kv_heads, n, dim, generator=gen).to(torch.bfloat16) for _ in range(2))
            cache.append_blocks(k.to(DEV), v.to(DEV))
            parts.append((k, v))
        dense.append([torch.from_numpy(kv4.quantized(torch.cat([p[i] for p in parts], 2)[0].double().numpy())) for i in (0, 1)])
    for cache, kv in zip(caches, dense):
        for got, want in zip(cache.as_tensors(), kv):
            assert got.dtype == torch.bfloat16 and torch.equal(got[0].double().cpu(), want)
    q = torch.randn(3, heads, 1, dim, generator=gen).to(torch.bfloat16).to(DEV)
    together = ar.full_attention_paged_batch(q, None, caches, config, runtime)
    for row, (cache, kv) in enumerate(zip(caches, dense)):
        n = kv[0].shape[1]
        want, mass = _attend(q[row].transpose(0, 1).double(), kv[0].to(DEV), kv[1].to(DEV), torch.ones(1, n, dtype=torch.bool, device=DEV), dim**-0.5)
        alone = ar.full_attention_paged(q[row : row + 1], None, cache, config, runtime)
        _close(together[row].transpose(0, 1), want, mass)
        _close(alone[0].transpose(0, 1), want, mass)
    assert runtime.paged_attention_stats.native_hits == 4
    other = FullAttentionCache(block_size=block, shared_pool=SharedKV4BlockPool(2, kv_heads, dim, block_size=block, device=DEV))
    other.append_blocks(torch.zeros(1, kv_heads, 1, dim, device=DEV), torch.zeros(1, kv_heads, 1, dim, device=DEV))
    assert ar.full_attention_paged_batch(q[:2], None, [caches[0], other], config, runtime) is None
    assert ar.full_attention_paged(q[:1].float(), None, caches[0], config, runtime) is None
    for cache in caches:
        cache.release()
    assert pool.free_blocks == list(range(24))


def test_steps_without_a_plan_are_refused_before_anything_is_written() -> None:
    heads, kv_heads, dim = 16, 2, 256
    config, runtime = _config(heads, kv_heads, dim), ar.HotPathRuntime()
    pool = SharedKV4BlockPool(8, kv_heads, dim, device=DEV)
    bf16 = SharedKVBlockPool(8, kv_heads, dim, device=DEV)
    tables = DeviceBatchPageTables(pool, rows=2, max_blocks=4)
    tables.add_request()
    x = lambda n: (torch.ones(n, heads * 2 * dim, dtype=torch.bfloat16, device=DEV), *(torch.ones(n, kv_heads * dim, dtype=torch.bfloat16, device=DEV) for _ in range(2)))  # noqa: E731
    w = [torch.zeros(dim, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    mrope = ar.RopeConfig(mrope_section=(11, 11, 10))
    for blocks, rope, kw in ((pool, ar.RopeConfig(), {}), (bf16, mrope, {}), (pool, mrope, dict(plan=tables.plan_step(), no_alloc=True))):
        with pytest.raises(ValueError, match="plan|no_alloc"):
            ar.full_attention_decode_step_device(*x(2), *w, blocks.key_blocks, blocks.value_blocks, tables, config, runtime, rope, **kw)
    at = torch.zeros(1, 2, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="positions"):
        ar.full_attention_decode_step_device(*x(2), *w, bf16.key_blocks, bf16.value_blocks, tables, config, runtime, plan=tables.plan_step(), positions=at)
    step = tables.reserve_prefill([0], [4])
    with pytest.raises(ValueError, match="positions"):
        ar.full_attention_prefill_device(*x(4), *w, bf16.key_blocks, bf16.value_blocks, step, config, runtime, positions=at)
    for blocks, rope in ((pool, ar.RopeConfig()), (bf16, mrope)):
        with pytest.raises(ValueError, match="plan_prefill"):
            ar.full_attention_prefill_device(*x(4), *w, blocks.key_blocks, blocks.value_blocks, step, config, runtime, rope)
    assert (pool.key_blocks == 0).all() and (bf16.key_blocks == 0).all()
    wide = replace(config, full_attention=replace(config.full_attention, num_heads=34))
    q = torch.ones(2, 34 * 2 * dim, dtype=torch.bfloat16, device=DEV)
    assert ar.full_attention_decode_step_device(q, *x(2)[1:], *w, pool.key_blocks, pool.value_blocks, tables, wide, runtime, plan=tables.plan_step()) is None
    assert runtime.paged_attention_stats.fallback_shape == 1
    # a step that does not fit: nothing taken, nothing written, zeros or nothing out
    tables.step_counts[0] = 5
    plan = tables.plan_step()
    with pytest.raises(RuntimeError, match="paged_kv_plan failed: more new tokens"):
        tables.check()
    assert (plan.slots == -1).all()


@pytest.mark.parametrize("dim,kv_heads", [(256, 2), (128, 4)])
def test_blocks_past_four_gigabytes(dim, kv_heads) -> None:
    """The same step in the first blocks of a pool and in blocks whose bytes lie past 2^32."""
    heads, block, rows = 8, 16, 2
    tile = hip_ops.kv4_tile_bytes(dim, block)
    blocks = (2**32 + 2**28) // (kv_heads * tile)
    pools = [torch.empty(blocks, kv_heads, tile, dtype=torch.uint8, device=DEV) for _ in range(2)]
    gen = torch.Generator().manual_seed(6)
    lens = [1500, 37]
    need = [-(-n // block) for n in lens]
    tokens = sum(lens)
    q, k, v = (torch.randn(tokens, h, dim, generator=gen).to(torch.bfloat16).to(DEV) for h in (2 * heads, kv_heads, kv_heads))
    q = q.view(tokens, heads, 2 * dim)
    w = torch.zeros(dim, dtype=torch.bfloat16, device=DEV)
    at = torch.cat([torch.arange(n) for n in lens]).to(DEV)
    cu = torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=torch.int32, device=DEV)
    results = []
    for first in (0, blocks - sum(need)):
        ids = first + torch.arange(sum(need), dtype=torch.int32, device=DEV)
        tables = torch.full((rows, max(need)), -1, dtype=torch.int32, device=DEV)
        tables[0, : need[0]], tables[1, : need[1]] = ids[: need[0]], ids[need[0] :]
        row = torch.repeat_interleave(torch.arange(rows, device=DEV), torch.tensor(lens, device=DEV))
        slots = tables[row, at // block].long() * block + at % block
        query, gate = hip_ops.qk_norm_mrope_kv_append(q, k, v, w, w, at, (dim // 4,), *pools, slots, block, eps=1e-6, rope_theta=1e6)
        prefill = hip_ops.paged_attention_prefill_kv4(query, cu, torch.zeros(rows, dtype=torch.int32, device=DEV), *pools, tables, block, max_new=max(lens), gate=gate)
        decode = hip_ops.paged_attention_decode_kv4(query[:rows].unsqueeze(2), tables, *pools, torch.tensor(lens, dtype=torch.int32, device=DEV), block)
        hip_ops.paged_kv4_append(k, v, *pools, slots, block)
        results.append((prefill, decode, *hip_ops.paged_kv4_gather(*pools, tables[:1], lens[0], block)))
    for low, high in zip(*results):
        assert torch.isfinite(low.float()).all() and torch.equal(low, high)


def test_two_streams_at_once() -> None:
    heads, kv_heads, dim, block = 16, 2, 256, 16
    pool = SharedKV4BlockPool(600, kv_heads, dim, block_size=block, device=DEV)
    gen = torch.Generator().manual_seed(7)
    k, v = (torch.randn(9600, kv_heads, dim, generator=gen).to(torch.bfloat16).to(DEV) for _ in range(2))
    hip_ops.paged_kv4_append(k, v, pool.key_blocks, pool.value_blocks, torch.randperm(9600, generator=gen).to(DEV), block)
    tables = torch.randperm(600, generator=gen)[:600].view(2, 300).to(DEV)
    q = torch.randn(2, heads, 1, dim, generator=gen).to(torch.bfloat16).to(DEV)
    new = torch.randn(40, heads, dim, generator=gen).to(torch.bfloat16).to(DEV)
    cu, prefix = torch.tensor([0, 15, 40], device=DEV), torch.tensor([4700, 3000], device=DEV)
    lens = [torch.tensor(n, device=DEV) for n in ([4800, 4000], [17, 4799])]
    runs = [lambda n=n: hip_ops.paged_attention_decode_kv4(q, tables, pool.key_blocks, pool.value_blocks, n, block) for n in lens]
    runs.append(lambda: hip_ops.paged_attention_prefill_kv4(new, cu, prefix, pool.key_blocks, pool.value_blocks, tables, block, max_new=25))
    want = [run() for run in runs]
    streams = [torch.cuda.Stream() for _ in runs]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for stream, run in zip(streams, runs):
            with torch.cuda.stream(stream):
                got.append(run())
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
