"""Prompts, decode steps and evictions together, as ``DensePagedCache`` and the serving backend run them."""
from types import SimpleNamespace as NS

import pytest
import torch

from test_dense_paged_gpu import evicted

pytestmark = pytest.mark.gpu
DEV = "cuda"


class Model:
    """The same steps in 64 bits: per layer and request, [H] lists of rows, weights and positions."""

    def __init__(self, layers, heads):
        self.heads, self.state = heads, [{} for _ in range(layers)]

    def attend(self, layer, request, q, k, v, scale, window=None):
        """q [n, Hq, D]; rows behind what is held.  Returns the output [n, Hq, D] and sum p |v|."""
        held = self.state[layer].setdefault(request, [[torch.zeros(0, k.shape[2], dtype=torch.float64, device=DEV)] * 2
                                                      + [torch.zeros(0, dtype=torch.float64, device=DEV), torch.zeros(0, dtype=torch.long, device=DEV), 0]
                                                      for _ in range(self.heads)])
        out, share, group, n = torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64), q.shape[1] // self.heads, q.shape[0]
        for h, (keys, values, w, pos, seen) in enumerate(held):
            keys, values = torch.cat([keys, k[:, h].double()]), torch.cat([values, v[:, h].double()])
            w, pos = torch.cat([w, w.new_zeros(n)]), torch.cat([pos, torch.arange(seen, seen + n, device=DEV)])
            sees = torch.arange(len(keys), device=DEV) <= len(keys) - n + torch.arange(n, device=DEV)[:, None]
            for g in range(h * group, (h + 1) * group):
                p = torch.softmax((q[:, g].double() @ keys.T * scale).masked_fill(~sees, -torch.inf), 1)
                out[:, g], share[:, g] = p @ values, p @ values.abs()
                w = w + p[-window if window else None:].sum(0)
            held[h] = [keys, values, w, pos, seen + n]
        return out, share


def close(got, want):
    """A probability and the result are rounded to bf16 once each; 2^-9 covers the logits, whose products of 128 fp32 sums
    are off by at most 128 2^-24 sum |q k| < 2^-10 here."""
    out, share = want
    u = 2.0 ** -8
    assert ((got.double() - out).abs() <= share * (u + 2.0 ** -9) + u * out.abs() * (1 + u) + 1e-30).all()


def rows(g, n, heads, dim):
    return torch.randn((n, heads, dim), generator=g, device=DEV).to(torch.bfloat16)


@pytest.mark.parametrize("heads,q_heads,dim,page,window", [(2, 14, 128, 16, None), (1, 4, 64, 24, 20)])
def test_prompts_decode_steps_and_evictions_together(heads, q_heads, dim, page, window):
    from inquant.dense_paged import DensePagedCache
    layers, g = 2, torch.Generator(device=DEV).manual_seed(1)
    cache = DensePagedCache(layers, heads, dim, pages=60, max_requests=4, max_tokens=600, page_tokens=page)
    model, scale = Model(layers, heads), dim ** -0.5

    def prompts(requests, tokens):
        step = cache.begin_prompt(requests, tokens)
        for layer in range(layers):
            q, k, v = rows(g, sum(tokens), q_heads, dim), rows(g, sum(tokens), heads, dim), rows(g, sum(tokens), heads, dim)
            out, at = step.attend(layer, q, k, v, window=window), 0
            for r, n in zip(requests, tokens):
                s = slice(at, at + n)
                close(out[s], model.attend(layer, r, q[s], k[s], v[s], scale, window))
                at += n
        step.finish()

    def decode(count):
        for _ in range(count):
            cache.begin_decode()
            for layer in range(layers):
                q, k, v = rows(g, 4, q_heads, dim), rows(g, 4, heads, dim), rows(g, 4, heads, dim)
                out = cache.decode(layer, q, k, v)
                used = {cache.slot(r): r for r in model.state[layer]}
                for slot in range(4):
                    if slot in used:
                        s = slice(slot, slot + 1)
                        close(out[s], model.attend(layer, used[slot], q[s], k[s], v[s], scale))
                    else:
                        assert (out[slot] == 0).all()
            cache.advance()

    def same_state(exact_weights=False):
        for layer in range(layers):
            for r, held in model.state[layer].items():
                k, v, pos = cache.gather(layer, r)
                assert k.shape[2] == cache.tokens(r) == len(held[0][0])
                for h in range(heads):
                    assert torch.equal(k[0, h].double(), held[h][0]) and torch.equal(v[0, h].double(), held[h][1]) and torch.equal(pos[h].long(), held[h][3])
                    w = cache.weights[layer, cache.slot(r), h, :k.shape[2]].double()
                    # a weight sums probabilities whose logits are off by less than 2^-10
                    assert ((w - held[h][2]).abs() <= 2.0 ** -9 * held[h][2] + 1e-12).all()

    def evict(budget, sink, recent):
        for layer in range(layers):
            for r, held in model.state[layer].items():
                for h in range(heads):
                    keys, values, w, pos, seen = held[h]
                    mine = cache.weights[layer, cache.slot(r), h].cpu()      # the same order of near-equal weights
                    o = torch.tensor(evicted(mine, pos.cpu(), len(keys), seen, budget, sink, recent), device=DEV)
                    held[h] = [keys[o], values[o], w[o], pos[o], seen]
        cache.evict(budget, sink=sink, recent=recent)

    for r in "abc":
        cache.admit(r)
    prompts(["c", "a", "b"], [130, 301, 7])
    decode(3)
    same_state()
    free = cache.free_pages
    evict(100, 4, 20)
    assert cache.free_pages > free and cache.tokens("a") == 100 and cache.tokens("b") == 10
    same_state()
    decode(page + 2)
    prompts(["b", "a"], [50, 33])                 # further chunks behind what is left
    cache.release("c")
    for layer in range(layers):
        del model.state[layer]["c"]
    cache.admit("d")
    prompts(["d"], [64])
    decode(2)
    same_state()
    evict(60, 0, 60)
    decode(1)
    same_state()
    from inquant import _native as N
    assert N.take_status(cache.device) == 0


def test_what_is_left_of_a_prompt_can_be_coded():
    from inquant.cache import CacheConfig, InQuantCache
    from inquant.codec import CodecConfig
    from inquant.dense_paged import DensePagedCache
    g = torch.Generator(device=DEV).manual_seed(2)
    cache = DensePagedCache(1, 4, 128, pages=80, max_requests=1, max_tokens=1200, page_tokens=16)
    cache.admit("a")
    step = cache.begin_prompt(["a"], [1000])
    step.attend(0, rows(g, 1000, 28, 128), rows(g, 1000, 4, 128), rows(g, 1000, 4, 128), window=64)
    step.finish()
    cache.evict(516, sink=4, recent=128)
    key, value, positions = cache.gather(0, "a")
    packed = InQuantCache(CacheConfig(CodecConfig(donor_policy="min_error"), block_size=128, residual_length=128, sink_tokens=4, value_bits=2,
                                      validate_positions=False))
    full_key, full_value = packed.update(key, value, 0)
    assert full_key.shape == key.shape and packed.get_seq_length(0) == 516 and len(packed._layers[0].key_blocks) > 0
    assert torch.equal(full_key[:, :, :4], key[:, :, :4]) and (positions[:, :4] == torch.arange(4, device=DEV)).all()


def test_captured_decode_steps_follow_the_cache():
    from inquant.dense_paged import DensePagedCache
    g = torch.Generator(device=DEV).manual_seed(3)
    caches = [DensePagedCache(2, 2, 128, pages=40, max_requests=2, max_tokens=300, page_tokens=16) for _ in range(2)]
    q, k, v = rows(g, 2, 14, 128), rows(g, 2, 2, 128), rows(g, 2, 2, 128)
    fill = [rows(g, 170, h, 128) for h in (14, 2, 2)]
    for c in caches:
        c.admit("a"), c.admit("b")
        step = c.begin_prompt(["a", "b"], [130, 40])
        for layer in range(2):
            step.attend(layer, *fill)
        step.finish()
        c.begin_decode()
    eager, captured = caches
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = [captured.decode(layer, q, k, v) for layer in range(2)]
    for i in range(40):
        q.copy_(rows(g, 2, 14, 128)), k.copy_(rows(g, 2, 2, 128)), v.copy_(rows(g, 2, 2, 128))
        want = [eager.decode(layer, q, k, v) for layer in range(2)]
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(want, outs))
        if i == 20:
            for c in caches:
                c.evict(96, sink=4, recent=30)
        for c in caches:
            c.advance() if i != 20 else None
            c.begin_decode()
    assert torch.equal(eager.positions, captured.positions) and torch.equal(eager.lengths, captured.lengths)


def test_prompts_of_a_step_attend_in_one_launch_of_the_backend(monkeypatch):
    import inquant_vllm.backend as backend
    from inquant.triton_attention import SharedDecodeWorkspace
    monkeypatch.setattr(backend, "WORKSPACE", SharedDecodeWorkspace())
    monkeypatch.setattr(backend, "get_current_vllm_config", lambda: NS(cache_config=NS(block_size=64), model_config=NS(max_model_len=512)))
    torch.manual_seed(4)
    lengths = {"a": 130, "b": 1, "c": 64, "d": 257}
    total = sum(lengths.values())
    q, k, v = (torch.randn(total, h, 128, dtype=torch.bfloat16, device=DEV) for h in (28, 4, 4))
    starts = [0]
    for n in lengths.values():
        starts.append(starts[-1] + n)
    tables = torch.randperm(24, device=DEV).to(torch.int32).view(4, 6)
    states, outs = [], []
    for batched in (False, True):
        impl = backend.InQuantImpl(28, 128, 128 ** -0.5, 4, None, None, "auto", max_requests=4)
        pool = torch.zeros((24, impl.layout.page_bytes), dtype=torch.uint8, device=DEV)
        out = torch.empty_like(q)
        metas = [backend.InQuantMetadata(n, n, 0, None, tables[i], name) for i, (name, n) in enumerate(lengths.items())]
        if batched:
            loc = torch.tensor(starts, dtype=torch.int32, device=DEV)
            assert impl.forward(None, q, k, v, pool, backend.InQuantPromptBatchMetadata(metas, loc), out) is out
        else:
            for m, at in zip(metas, starts):
                s = slice(at, at + m.num_actual_tokens)
                impl.forward(None, q[s], k[s], v[s], pool, m, out[s])
        states.append((impl, pool))
        outs.append(out)
    (one, pool1), (many, pool2) = states
    assert torch.equal(pool1, pool2) and one.prefill_calls == many.prefill_calls == 4
    for name, n in lengths.items():
        a, b = one.requests[name], many.requests[name]
        assert (a.tokens, a.sealed_pages) == (b.tokens, b.sealed_pages) == (n, n // 64)
        for first, count in ((0, min(4, n)), (4, n % 64)):
            assert torch.equal(a.dense[:, :, first:first + count], b.dense[:, :, first:first + count])
    # two kernels, each within a rounding of its probabilities and one of its result
    assert (outs[0].float() - outs[1].float()).abs().max() <= 4 * 2.0 ** -8 * v.abs().max().float()
    meta = backend.InQuantMetadata(1, lengths["a"] + 1, lengths["a"], None, tables[0], "a")
    impl = many
    with pytest.raises(RuntimeError, match="without context"):
        impl.forward(None, q, k, v, pool2, backend.InQuantPromptBatchMetadata([meta], torch.tensor([0, 1], dtype=torch.int32, device=DEV)), outs[0])
    fresh = [backend.InQuantMetadata(1, 1, 0, None, tables[0], r) for r in "vwxyz"]
    with pytest.raises(RuntimeError, match="max_requests"):
        impl.forward(None, q, k, v, pool2, backend.InQuantPromptBatchMetadata(fresh, torch.arange(6, dtype=torch.int32, device=DEV)), outs[0])
    with pytest.raises(ValueError, match="query_start_loc"):
        impl.forward(None, q, k, v, pool2, backend.InQuantPromptBatchMetadata(fresh[:2], None), outs[0])
    assert set(impl.requests) == set(lengths)
