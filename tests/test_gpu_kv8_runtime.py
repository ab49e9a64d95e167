"""The operators run together on 8-bit pools: prompts in chunks, decode steps, a request forked into several answers, requests
freed on the device, the cache compacted, a replayed graph; and forks on bf16 and 4-bit pools."""

from __future__ import annotations

import pytest
import torch

import attention_runtime as ar
import hip_ops
from decode_state import DeviceBatchPageTables, FullAttentionCache, LinearStatePool, SharedKV4BlockPool, SharedKV8BlockPool, SharedKVBlockPool
from test_gpu_attention_kv8 import _attend, _close

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _config(heads, kv_heads, dim, gate=True):
    text = {"linear_num_key_heads": 1, "linear_num_value_heads": 1, "linear_key_head_dim": 4, "linear_value_head_dim": 4, "linear_conv_kernel_dim": 4,
            "num_attention_heads": heads, "num_key_value_heads": kv_heads, "head_dim": dim, "attn_output_gate": gate, "native_paged_attention": True}
    return ar.parse_attention_config({"text_config": text})


class _Layer:
    """One layer of a running batch.  Each request has a pool of its own beside it, written by the same calls: what the batch's
    pool has to hold for it."""

    def __init__(self, seed, pool, heads, kv_heads, dim, rope, most):
        self.gen = torch.Generator().manual_seed(seed)
        self.pool, self.heads, self.kv_heads, self.dim, self.rope = pool, heads, kv_heads, dim, rope
        self.qw, self.kw = (self._bf(dim) * 0.3 for _ in range(2))
        self.blocks = -(-most // pool.block_size)
        self.beside = {}  # request -> (key pool, value pool, tokens)

    def _bf(self, *shape):
        return torch.randn(*shape, generator=self.gen).to(torch.bfloat16).to(DEV)

    def tokens(self, n):
        scale = torch.exp(torch.randn(n, 1, generator=self.gen)).to(torch.bfloat16).to(DEV)  # values whose runs grow
        return self._bf(n, self.heads * 2 * self.dim), self._bf(n, self.kv_heads * self.dim), self._bf(n, self.kv_heads * self.dim) * scale

    def took(self, req, q, k, v, positions):
        """The request's new tokens go to its own pool; their queries."""
        n = q.shape[0]
        if req not in self.beside:
            pool = SharedKV8BlockPool(self.blocks, self.kv_heads, self.dim, block_size=self.pool.block_size, device=DEV)
            self.beside[req] = pool.key_blocks, pool.value_blocks, 0
        keys, values, length = self.beside[req]
        kb, vb = (torch.zeros(-(-n // 16), self.kv_heads, 16, self.dim, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        query, _ = hip_ops.qk_norm_mrope_kv_append(q, k, v, self.qw, self.kw, positions, self.rope.sections(self.dim), kb, vb, torch.arange(n, device=DEV), 16,
                                                   eps=self.rope.rms_norm_eps, rope_theta=self.rope.rope_theta, interleaved=self.rope.mrope_interleaved)
        rows = [x.transpose(1, 2).reshape(-1, self.kv_heads, self.dim)[:n] for x in (kb, vb)]
        hip_ops.paged_kv8_append(*rows, keys, values, torch.arange(length, length + n, device=DEV), self.pool.block_size)
        self.beside[req] = keys, values, length + n
        return query

    def forked(self, req, child):
        keys, values, length = self.beside[req]
        self.beside[child] = keys.clone(), values.clone(), length

    def check(self, req, q, k, v, positions, out, table):
        query = self.took(req, q, k, v, positions)
        own_keys, own_values, total = self.beside[req]
        n, block = q.shape[0], self.pool.block_size
        want_kv = hip_ops.paged_kv8_gather(own_keys, own_values, torch.arange(self.blocks, device=DEV), total, block)
        got_kv = hip_ops.paged_kv8_gather(self.pool.key_blocks, self.pool.value_blocks, table.unsqueeze(0).contiguous(), total, block)
        assert torch.equal(got_kv[0], want_kv[0]) and torch.equal(got_kv[1], want_kv[1]), req
        seen = torch.arange(total, device=DEV) <= torch.arange(total - n, total, device=DEV).unsqueeze(1)
        want, mass = _attend(query.double(), want_kv[0][0].double(), want_kv[1][0].double(), seen, self.dim**-0.5)
        _close(out.view(n, self.heads, self.dim), want, mass, q.view(n, self.heads, 2 * self.dim)[..., self.dim:])


@pytest.mark.parametrize("heads,kv_heads,dim,block,sections,interleaved", [(16, 2, 256, 16, (11, 11, 10), True), (20, 4, 128, 32, (16, 24, 24), False), (8, 8, 128, 16, None, False)])
def test_a_running_batch(heads, kv_heads, dim, block, sections, interleaved) -> None:
    rope = ar.RopeConfig(rope_theta=1e6, mrope_section=sections, mrope_interleaved=interleaved)
    config, runtime = _config(heads, kv_heads, dim), ar.HotPathRuntime()
    layers = [_Layer(seed, SharedKV8BlockPool(60, kv_heads, dim, block_size=block, device=DEV), heads, kv_heads, dim, rope, 8 * block) for seed in (1, 2)]
    tables = DeviceBatchPageTables(layers[0].pool, rows=9, max_blocks=8)
    pools = [t for layer in layers for t in (layer.pool.key_blocks, layer.pool.value_blocks)]
    axes = len(rope.sections(dim))
    length, row_of = {}, {}

    def spread(places):
        return torch.tensor(places, device=DEV).expand(axes, -1).contiguous()

    def chunk(counts):
        reqs = sorted(counts, key=row_of.get)
        step = tables.plan_prefill([row_of[r] for r in reqs], [counts[r] for r in reqs])
        positions = spread([length[r] + i for r in reqs for i in range(counts[r])])
        for layer in layers:
            q, k, v = layer.tokens(positions.shape[1])
            out = ar.full_attention_prefill_device(q, k, v, layer.qw, layer.kw, layer.pool.key_blocks, layer.pool.value_blocks, step, config, runtime, rope)
            at = 0
            for r in reqs:
                part = slice(at, at + counts[r])
                at += counts[r]
                layer.check(r, q[part], k[part], v[part], positions[:, part], out[part], tables.block_tables[row_of[r]])
        for r in reqs:
            length[r] += counts[r]

    def decode(inputs):
        plan = tables.plan_step()
        return [ar.full_attention_decode_step_device(*x, layer.qw, layer.kw, layer.pool.key_blocks, layer.pool.value_blocks, tables, config, runtime, rope, plan=plan)
                for layer, x in zip(layers, inputs)]

    def check_step(inputs, outs):
        for layer, (q, k, v), out in zip(layers, inputs, outs):
            for r, row in row_of.items():
                one = slice(row, row + 1)
                layer.check(r, q[one], k[one], v[one], spread([length[r]]), out[one], tables.block_tables[row])
            for row in set(range(tables.rows)) - set(row_of.values()):
                assert (out[row] == 0).all()
        for r in row_of:
            length[r] += 1

    def step():
        inputs = [layer.tokens(tables.rows) for layer in layers]
        check_step(inputs, decode(inputs))
        tables.check()

    for req in "abc":
        row_of[req], length[req] = tables.add_request(), 0
    chunk({"a": 20, "b": 5, "c": 2 * block})
    step()
    chunk({"a": 17, "b": 30})
    for parent, children in (("a", "de"), ("c", "f")):
        for child, row in zip(children, tables.fork_request(row_of[parent], len(children), pools)):
            row_of[child], length[child] = row, length[parent]
            for layer in layers:
                layer.forked(parent, child)
    shared = length["a"] // block
    assert torch.equal(tables.block_tables[row_of["d"], :shared], tables.block_tables[row_of["a"], :shared])
    assert tables.block_tables[row_of["d"], shared] != tables.block_tables[row_of["a"], shared]
    step()
    step()
    free = tables.allocator.free_count
    tables.release_requests([row_of.pop("a"), row_of.pop("b")])  # what d and e share of a stays
    assert tables.allocator.free_count > free
    step()
    tables.release_request(row_of.pop("d"))
    tables.compact(pools)
    used = sorted({b for row in tables.block_tables.tolist() for b in row if b >= 0})
    assert used == list(range(len(used)))
    step()
    chunk({"e": 3, "f": 18})
    row_of["g"], length["g"] = tables.add_request(), 0
    chunk({"g": 19})
    tables.compact(pools, max_moves=1)
    step()
    inputs = [layer.tokens(tables.rows) for layer in layers]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        outs = decode(inputs)
    for _ in range(3):
        for layer, x in zip(layers, inputs):
            for old, new in zip(x, layer.tokens(tables.rows)):
                old.copy_(new)
        graph.replay()
        check_step([[t.clone() for t in x] for x in inputs], outs)
        tables.check()
    tables.release_requests([row_of.pop(r) for r in list(row_of)])
    assert tables.allocator.free_count == 60 and not tables.allocator.references.any()
    assert runtime.paged_attention_stats.dense_fallbacks == 0


def test_slots_of_a_step_whose_first_call_is_captured() -> None:
    ar._COUNT_UP.clear()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        inside = ar._count_up(11, torch.device(DEV)) + 0
    want = torch.arange(11, device=DEV)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        eager = [ar._count_up(n, torch.device(DEV)) + 0 for n in (11, 9, 16)]
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(inside, want) and torch.equal(eager[0], want) and torch.equal(eager[1], want[:9]) and eager[2].shape == (16,)


def test_post_rotary_keys_and_values_on_an_8_bit_pool() -> None:
    heads, kv_heads, dim, block, rows = 16, 2, 256, 16, 3
    config, runtime = _config(heads, kv_heads, dim), ar.HotPathRuntime()
    pool = SharedKV8BlockPool(8, kv_heads, dim, block_size=block, device=DEV)
    tables = DeviceBatchPageTables(pool, rows=rows, max_blocks=4)
    tables.add_request()
    tables.add_request()
    gen = torch.Generator().manual_seed(4)
    for i in range(3):
        bf = lambda *shape: torch.randn(*shape, generator=gen).to(torch.bfloat16).to(DEV)  # noqa: E731
        q, k, v, gate = bf(rows, heads, 1, dim), bf(rows, kv_heads, 1, dim), bf(rows, kv_heads, 1, dim), bf(rows, 1, heads * dim)
        plan = tables.plan_step()
        out = ar.full_attention_decode_device(q, gate, k, v, pool.key_blocks, pool.value_blocks, tables, config, runtime, plan=plan)
        for row in (0, 1):
            keys, values = hip_ops.paged_kv8_gather(pool.key_blocks, pool.value_blocks, tables.block_tables[row], i + 1, block)
            # the newest token is off by half a step of its codes at most: 2^-4 of it, and half a step below the least normal one
            assert ((keys[0, :, i] - k[row, :, 0]).abs() <= 2.0**-4 * k[row, :, 0].abs() + 2.0**-17 * k[row].abs().max()).all()
            want, mass = _attend(q[row].transpose(0, 1).double(), keys[0].double(), values[0].double(), torch.ones(1, i + 1, dtype=torch.bool, device=DEV), dim**-0.5)
            s = torch.sigmoid(gate[row].double()).view(1, heads, dim)
            got = out[row].view(1, heads, dim).double()
            # the heads, the sigmoid and their product are rounded to bf16, the probabilities too
            assert ((got - want * s).abs() <= 2.0**-8 * (3.05 * (want * s).abs() + mass * s) + 2.0**-10 * mass * s).all()
        assert not out[2].any()
    with pytest.raises(ValueError, match="plan"):
        ar.full_attention_decode_device(q, gate, k, v, pool.key_blocks, pool.value_blocks, tables, config, runtime)
    with pytest.raises(ValueError, match="no_alloc"):
        ar.full_attention_decode_device(q, gate, k, v, pool.key_blocks, pool.value_blocks, tables, config, runtime, plan=plan, no_alloc=True)


def test_caches_of_single_requests_on_an_8_bit_pool() -> None:
    heads, kv_heads, dim = 8, 2, 128
    config, runtime = _config(heads, kv_heads, dim, gate=False), ar.HotPathRuntime()
    pool = SharedKV8BlockPool(20, kv_heads, dim, device=DEV)
    caches = [FullAttentionCache(shared_pool=pool) for _ in range(2)]
    gen = torch.Generator().manual_seed(5)
    for cache, chunks in zip(caches, ((5, 30, 1), (16, 1, 1, 9))):
        for n in chunks:
            k, v = (torch.randn(1, kv_heads, n, dim, generator=gen).to(torch.bfloat16).to(DEV) for _ in range(2))
            cache.append_blocks(k, v)
    query = torch.randn(2, heads, 1, dim, generator=gen).to(torch.bfloat16).to(DEV)
    both = ar.full_attention_paged_batch(query, None, caches, config, runtime)
    for row, cache in enumerate(caches):
        keys, values = cache.as_tensors()
        assert keys.shape == (1, kv_heads, cache.valid, dim)
        want, mass = _attend(query[row].transpose(0, 1).double(), keys[0].double(), values[0].double(), torch.ones(1, cache.valid, dtype=torch.bool, device=DEV), dim**-0.5)
        _close(both[row].transpose(0, 1), want, mass)
        one = ar.full_attention_paged(query[row : row + 1], None, cache, config, runtime)
        _close(one[0].transpose(0, 1), want, mass)
        cache.release()
    assert len(pool.free_blocks) == 20 and runtime.paged_attention_stats.dense_fallbacks == 0


@pytest.mark.parametrize("kind", ["bf16", "4-bit"])
def test_forks_on_other_pools(kind) -> None:
    """A fork's rows read what their source holds, and what each writes stays its own."""
    heads, kv_heads, dim = 16, 2, 256
    config, runtime = _config(heads, kv_heads, dim), ar.HotPathRuntime()
    pool = (SharedKVBlockPool if kind == "bf16" else SharedKV4BlockPool)(30, kv_heads, dim, device=DEV)
    tables = DeviceBatchPageTables(pool, rows=4, max_blocks=6)
    pools = [pool.key_blocks, pool.value_blocks]
    gen = torch.Generator().manual_seed(6)
    bf = lambda *shape: torch.randn(*shape, generator=gen).to(torch.bfloat16).to(DEV)  # noqa: E731
    weights = bf(dim) * 0.3, bf(dim) * 0.3
    row = tables.add_request()
    step = tables.plan_prefill([row], [37])
    ar.full_attention_prefill_device(bf(37, heads * 2 * dim), bf(37, kv_heads * dim), bf(37, kv_heads * dim), *weights, *pools, step, config, runtime, ar.RopeConfig(mrope_section=(11, 11, 10)))
    children = tables.fork_request(row, 2, pools)
    assert children == [1, 2] and tables.sequence_lengths.tolist() == [37, 37, 37, 0]
    x = [bf(1, heads * 2 * dim), bf(1, kv_heads * dim), bf(1, kv_heads * dim)]
    same = [t.expand(4, -1).contiguous() for t in x]
    decode = lambda inputs: ar.full_attention_decode_step_device(*inputs, *weights, *pools, tables, config, runtime, ar.RopeConfig(mrope_section=(11, 11, 10)), plan=tables.plan_step())  # noqa: E731
    out = decode(same)
    assert torch.equal(out[0], out[1]) and torch.equal(out[0], out[2]) and not out[3].any()
    other = [t.clone() for t in same]
    other[1][1] += 1
    out = decode(other)
    assert torch.equal(out[0], out[2]) and not torch.equal(out[0], out[1])
    tables.compact(pools)
    out = decode(same)
    assert torch.equal(out[0], out[2]) and not torch.equal(out[0], out[1])
    tables.release_requests([0, 1, 2])
    assert tables.allocator.free_count == 30


def test_a_fork_without_blocks_takes_nothing() -> None:
    pool = SharedKV8BlockPool(4, 2, 128, device=DEV)
    tables = DeviceBatchPageTables(pool, rows=6, max_blocks=4)
    tables.add_request(prompt_tokens=40)  # two blocks and a half
    with pytest.raises(RuntimeError, match="paged_kv_fork failed: shared KV pool exhausted"):
        tables.fork_request(0, 2, [pool.key_blocks, pool.value_blocks])
    assert tables.active == [True] + [False] * 5 and tables.allocator.free_count == 1 and not tables.allocator.references.any()
    assert tables.fork_request(0, 1, [pool.key_blocks, pool.value_blocks]) == [1]
    assert tables.step_counts.tolist() == [1, 1, 0, 0, 0, 0]


def test_forks_of_recurrent_states() -> None:
    pool = LinearStatePool(6, 2, 128, 128, 24, 4, device=DEV)
    slot = pool.acquire()
    pool.state[slot].normal_()
    pool.conv[slot].normal_()
    taken = pool.fork(slot, 3)
    assert taken == [1, 2, 3] and pool.free_slots == [4, 5]
    for t in taken:
        assert torch.equal(pool.state[t], pool.state[slot]) and torch.equal(pool.conv[t], pool.conv[slot])
    assert not pool.state[4:].any()
