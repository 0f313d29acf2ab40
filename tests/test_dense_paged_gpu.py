"""Decode over uncompressed pages and eviction (``inquant.dense_paged``) against their formulas in 64 bits.

Bounds.  u is half a step of the dtype.  A logit's fp32 error is at most delta = D 2^-24 scale sum |q_c k_c|, the relative
error of its exponential; 2^-20 covers the exponential unit, the factors of the joins and fp32 sums in chains of a few
hundred.  A probability is rounded to the dtype once (u) before the product with the values, its normaliser is
not (2 delta for both), the result is rounded once: |out - exact| <= sum p |v| (u + 2 delta) + u |exact| (1 + u).  A
weight is a sum of unrounded probabilities: 2 delta of it, and a step of the accumulated sum."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


class Pool:
    """A paged cache with the given lengths, its pages in random order and what no token fills not a number."""

    def __init__(self, lengths, heads, dim, page, dtype, seed=0, spare=0, columns=None):
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.lengths, self.page = lengths, page
        need = [max(1, -(-(max(n, 0) + 1) // page)) for n in lengths]
        self.columns = columns or max(need) + spare
        ids = torch.randperm(sum(need) + 2, generator=g, device=DEV).to(torch.int32)
        self.table = torch.full((len(lengths), self.columns), -5, dtype=torch.int32, device=DEV)     # unused entries are nobody's
        self.keys = torch.full((sum(need) + 2, heads, page, dim), float("nan"), dtype=dtype, device=DEV)
        self.values = self.keys.clone()
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = ids[at:at + n]
            at += n
            if lengths[b] > 0:
                k, v = (torch.randn((lengths[b], heads, dim), generator=g, device=DEV).to(dtype) for _ in range(2))
                self.put(b, torch.arange(lengths[b], device=DEV), k, v)
        self.n = ints(lengths)

    def places(self, b, tokens):
        return self.table[b].long()[tokens // self.page], tokens % self.page

    def put(self, b, tokens, k, v):
        p, o = self.places(b, tokens)
        self.keys[p, :, o], self.values[p, :, o] = k, v

    def get(self, b, count):
        p, o = self.places(b, torch.arange(count, device=DEV))
        return self.keys[p, :, o], self.values[p, :, o]


def check_token(pool, q, got, weights=None, old=None, fresh=None, scale=None, tokens=None):
    """Compares output (and accumulated weights) with the formula over what the pool holds now."""
    u, dim = torch.finfo(q.dtype).eps / 2, q.shape[2]
    scale = dim ** -0.5 if scale is None else scale
    heads, group = pool.keys.shape[1], q.shape[1] // pool.keys.shape[1]
    for b, n in enumerate(tokens if tokens is not None else [max(n, 0) + (fresh is not None and n >= 0) for n in pool.lengths]):
        if n == 0:
            assert (got[b] == 0).all()
            continue
        k, v = (t.double().transpose(0, 1) for t in pool.get(b, n))
        x = q[b].double().reshape(heads, group, dim)
        logits = x @ k.transpose(1, 2) * scale
        delta = dim * 2.0 ** -24 * scale * (x.abs() @ k.abs().transpose(1, 2)).amax(2, keepdim=True) + 2.0 ** -20
        p = torch.softmax(logits, 2)
        want, share = (p @ v).reshape(-1, dim), (p @ v.abs()).reshape(-1, dim)
        allowed = share * (u + 2 * delta.reshape(-1, 1)) + u * want.abs() * (1 + u) + torch.finfo(q.dtype).smallest_normal
        off = (got[b].double() - want).abs()
        assert (off <= allowed).all(), (b, n, (off / allowed).max())
        if weights is not None:
            step = p.sum(1)
            before = torch.zeros_like(step) if old is None else old[b, :, :n].double().clone()
            if fresh is not None and old is not None:
                before[:, n - 1] = 0
            allowed = (p * 2 * delta).sum(1) + (group + 1) * 2.0 ** -24 * (step + before)
            assert ((weights[b, :, :n].double() - step - before).abs() <= allowed).all()


def query(requests, q_heads, dim, dtype, seed=7):
    return torch.randn((requests, q_heads, dim), generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


SHAPES = [(28, 4, 128, torch.bfloat16), (12, 1, 128, torch.float16), (8, 8, 64, torch.float16), (40, 2, 64, torch.bfloat16),
          (20, 1, 128, torch.bfloat16)]


@pytest.mark.parametrize("q_heads,heads,dim,dtype", SHAPES)
@pytest.mark.parametrize("page", [1, 16, 24, 256])
@pytest.mark.parametrize("lengths", [[1], [15, 16, 17], [127, 128, 129, 0, 1], [700, -1, 2500, 3]])
def test_tokens_over_pages(q_heads, heads, dim, dtype, page, lengths):
    from inquant.dense_paged import paged_attention
    pool = Pool(lengths, heads, dim, page, dtype)
    q = query(len(lengths), q_heads, dim, dtype)
    kept = pool.keys.clone(), pool.values.clone()
    out = paged_attention(q, pool.keys, pool.values, pool.table, pool.n)
    check_token(pool, q, out)
    assert torch.equal(pool.keys.view(torch.int16), kept[0].view(torch.int16)) and torch.equal(pool.values.view(torch.int16), kept[1].view(torch.int16))


@pytest.mark.parametrize("q_heads,heads,dim,dtype", SHAPES)
@pytest.mark.parametrize("page", [16, 24, 64])
@pytest.mark.parametrize("lengths", [[0], [0, 1, 127, 128], [-1, 300, 0, 1111]])
def test_new_tokens_are_stored_and_weights_kept_up(q_heads, heads, dim, dtype, page, lengths):
    from inquant.dense_paged import paged_attention
    pool = Pool(lengths, heads, dim, page, dtype, seed=1, spare=1)
    q = query(len(lengths), q_heads, dim, dtype)
    new_k, new_v = query(len(lengths), heads, dim, dtype, 8), query(len(lengths), heads, dim, dtype, 9)
    width = pool.columns * page
    old = torch.rand((len(lengths), heads, width + 3), device=DEV)
    before = pool.keys.clone()
    into = torch.full((len(lengths), heads, width), 5.0, device=DEV)
    out, w = paged_attention(q, pool.keys, pool.values, pool.table, pool.n, new_key=new_k, new_value=new_v, weights=old, out_weights=into)
    assert w is into
    for b, n in enumerate(lengths):
        if n >= 0:
            k, v = pool.get(b, n + 1)
            assert torch.equal(k[n], new_k[b]) and torch.equal(v[n], new_v[b])
            p, o = pool.places(b, torch.tensor([n], device=DEV))
            before[p, :, o] = new_k[b]
        assert (into[b, :, max(n + 1, 0):] == 5.0).all()
    assert torch.equal(before.view(torch.int16), pool.keys.view(torch.int16))      # nothing else was written
    check_token(pool, q, out, w, old, fresh=True)
    # in place, and this step's weights alone
    again = old.clone()
    out2, w2 = paged_attention(q, pool.keys, pool.values, pool.table, pool.n, new_key=new_k, new_value=new_v, weights=again)
    assert w2 is again and torch.equal(out2, out)
    for b, n in enumerate(lengths):
        assert torch.equal(again[b, :, :max(n + 1, 0)], into[b, :, :max(n + 1, 0)])
    _, alone = paged_attention(q, pool.keys, pool.values, pool.table, pool.n, new_key=new_k, new_value=new_v, out_weights=into)
    check_token(pool, q, out, alone, None, fresh=True)


@pytest.mark.parametrize("lengths", [[40000], [1] * 300 + [5000], [0] * 40 + [130] * 40])
def test_many_parts_and_many_requests(lengths):
    from inquant.dense_paged import paged_attention
    pool = Pool(lengths, 2, 128, 16, torch.bfloat16, seed=2)
    q = query(len(lengths), 14, 128, torch.bfloat16)
    weights = torch.zeros((len(lengths), 2, pool.columns * 16), device=DEV)
    out, w = paged_attention(q, pool.keys, pool.values, pool.table, pool.n, out_weights=weights)
    check_token(pool, q, out, w)
    assert torch.equal(out, paged_attention(q, pool.keys, pool.values, pool.table, pool.n))


def test_large_logits_and_rising_maxima():
    from inquant.dense_paged import paged_attention
    pool = Pool([3000], 2, 128, 16, torch.bfloat16, seed=3)
    p, o = pool.places(0, torch.arange(3000, device=DEV))
    pool.keys[p, :, o] *= torch.linspace(0.1, 8, 3000, device=DEV)[:, None, None].to(torch.bfloat16)
    q = query(1, 8, 128, torch.bfloat16) * 2
    check_token(pool, q, paged_attention(q, pool.keys, pool.values, pool.table, pool.n))


def test_strides_of_pages_and_rows():
    from inquant.dense_paged import paged_attention
    lengths = [300, 77]
    pool = Pool(lengths, 2, 128, 16, torch.bfloat16, seed=4)
    q = query(2, 8, 128, torch.bfloat16)
    new_k, new_v = query(2, 2, 128, torch.bfloat16, 8), query(2, 2, 128, torch.bfloat16, 9)
    want = paged_attention(q, pool.keys.clone(), pool.values.clone(), pool.table, pool.n, new_key=new_k, new_value=new_v)
    both = torch.empty((pool.keys.shape[0], 2, 16, 2, 128), dtype=q.dtype, device=DEV)       # token-major, K beside V
    keys, values = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    keys.copy_(pool.keys), values.copy_(pool.values)
    table = torch.full((2, pool.columns + 5), -9, dtype=torch.int32, device=DEV)
    table[:, :pool.columns] = pool.table
    for shift in (0, 3):      # query and new rows that do not start on 16 bytes are copied
        x, nk, nv = (torch.empty(t.numel() + shift, dtype=t.dtype, device=DEV)[shift:].view(t.shape).copy_(t) for t in (q, new_k, new_v))
        room = torch.empty((2, 8, 256), dtype=q.dtype, device=DEV)[:, :, 128:]
        got = paged_attention(x, keys, values, table[:, :pool.columns], pool.n.repeat_interleave(2)[::2], new_key=nk, new_value=nv, out=room)
        assert got is room and torch.equal(got, want)


def test_pages_and_lengths_out_of_range():
    from inquant import _native as N
    from inquant.dense_paged import paged_attention
    lengths = [200, 40]
    pool = Pool(lengths, 2, 128, 16, torch.bfloat16, seed=5)
    q = query(2, 4, 128, torch.bfloat16)
    new = query(2, 2, 128, torch.bfloat16, 8)
    assert N.take_status(q.device) == 0
    want = paged_attention(q, pool.keys, pool.values, pool.table, pool.n)
    for bad in (-1, pool.keys.shape[0], 2 ** 31 - 1):
        table = pool.table.clone()
        table[0, 3:6] = bad       # tokens 48 .. 95 are left out
        weights = torch.full((2, 2, pool.columns * 16), 7.0, device=DEV)
        out, w = paged_attention(q, pool.keys, pool.values, table, pool.n, out_weights=weights)
        assert N.take_status(q.device) == N.STATUS_BAD_INDEX
        assert torch.equal(out[1], want[1]) and (w[0, :, 48:96] == 0).all() and torch.isfinite(out).all()
        k, v = pool.get(0, 200)
        rest = torch.cat([torch.arange(48), torch.arange(96, 200)]).to(DEV)
        p = torch.softmax(q[0].double().view(2, 2, 128) @ k[rest].double().permute(1, 2, 0) * 128 ** -0.5, 2)
        assert ((p @ v[rest].double().transpose(0, 1)).view(4, 128) - out[0].double()).abs().max() < 2.0 ** -7
    # a table that has no room for the new token, a length beyond it: nothing is stored, the table's tokens are attended to
    short = pool.table[:, :2].contiguous()
    keys = pool.keys.clone()
    full = paged_attention(q, pool.keys, pool.values, short, ints([32, 32]))
    for n in (32, 100, 2 ** 31 - 1):
        out = paged_attention(q, pool.keys, pool.values, short, ints([n, 32]), new_key=new, new_value=new)
        assert N.take_status(q.device) == N.STATUS_BAD_INDEX and torch.equal(out, full)
    assert torch.equal(keys.view(torch.int16), pool.keys.view(torch.int16))
    # a place for the new token in a page that is not there
    table = pool.table.clone()
    table[0, 12] = -1             # tokens 192 .. 207
    out = paged_attention(q, pool.keys, pool.values, table, pool.n, new_key=new, new_value=new)
    assert N.take_status(q.device) == N.STATUS_BAD_INDEX and torch.isfinite(out).all()
    assert torch.equal(keys.view(torch.int16)[pool.table[0, 12].long()], pool.keys.view(torch.int16)[pool.table[0, 12].long()])


def test_captured_steps_follow_lengths_and_share_no_scratch():
    from inquant.dense_paged import paged_attention
    lengths = [100, 900]
    pool = Pool(lengths, 4, 128, 16, torch.bfloat16, seed=6, spare=4)
    q = query(2, 28, 128, torch.bfloat16)
    n = ints(lengths)
    weights = torch.zeros((2, 4, pool.columns * 16), device=DEV)
    graphs = []
    for _ in range(2):
        stream = torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = paged_attention(q, pool.keys, pool.values, pool.table, n, out_weights=torch.zeros_like(weights))
        graphs.append((graph, got, stream))
    for mix in ([100, 900], [1, 33], [0, -1], [64, 800]):
        n.copy_(ints(mix))
        want = paged_attention(q, pool.keys, pool.values, pool.table, ints(mix), out_weights=torch.zeros_like(weights))
        torch.cuda.synchronize()
        for graph, _, stream in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for _, got, _ in graphs:
            assert torch.equal(got[0], want[0])
            for b in range(2):
                assert torch.equal(got[1][b, :, :max(mix[b], 0)], want[1][b, :, :max(mix[b], 0)])


def test_a_long_cache_whose_offsets_pass_32_bits():
    """Pages behind 2^31 elements of a pool that shares its storage with other data."""
    from inquant.dense_paged import paged_attention
    lengths = [500]
    pool = Pool(lengths, 2, 128, 16, torch.bfloat16, seed=7)
    wide = torch.empty(2 ** 31 + 40 * 4096, dtype=torch.bfloat16, device=DEV)
    count = pool.keys.shape[0]
    keys = wide.as_strided((count, 2, 16, 128), (2 ** 31 // count // 8 * 8, 2048, 128, 1))
    keys.copy_(pool.keys)
    q = query(1, 14, 128, torch.bfloat16)
    assert torch.equal(paged_attention(q, keys, pool.values, pool.table, pool.n), paged_attention(q, pool.keys, pool.values, pool.table, pool.n))


# ------------------------------------------------------------------------------------------------ eviction
def evicted(weights, positions, length, seen, budget, sink, recent):
    """Places (origin of what lies at each of the first min(length, budget) places) of one row, from the definition."""
    w = [(-math.inf if math.isnan(x) else x) for x in weights[:length].tolist()]
    nan = [math.isnan(x) for x in weights[:length].tolist()]
    p = positions[:length].tolist()
    if length <= budget:
        return list(range(length))
    safe = [p[j] < sink or p[j] >= seen - recent for j in range(length)]
    order = sorted(range(length), key=lambda j: (not safe[j], not safe[j] and nan[j], 0.0 if safe[j] else -w[j], j))
    kept = set(order[:budget])
    free = [j for j in range(budget) if j not in kept]
    moving = [j for j in range(budget, length) if j in kept]
    origin = list(range(budget))
    for to, source in zip(free, moving):
        origin[to] = source
    return origin


def check_evict(pool, heads, lengths, seen, weights, positions, budget, sink, recent, in_place=False):
    from inquant.dense_paged import evict_tokens
    keys, values = pool.keys.clone(), pool.values.clone()
    want = [[evicted(weights[b, h].cpu(), positions[b, h].cpu(), max(n, 0), seen[b], budget, sink, recent) for h in range(heads)]
            for b, n in enumerate(lengths)]
    w0, p0, n0 = weights.clone(), positions.clone(), ints(lengths)
    into = dict(out_weights=weights, out_positions=positions, out_lengths=n0) if in_place else {}
    if in_place == "state":
        del into["out_lengths"]
    n, w, p = evict_tokens(pool.keys, pool.values, pool.table, n0, weights, positions, ints(seen), budget, sink=sink, recent=recent, **into)
    assert n.tolist() == [min(x, budget) for x in lengths]
    for b in range(len(lengths)):
        for h in range(heads):
            o = torch.tensor(want[b][h], dtype=torch.long, device=DEV)
            assert torch.equal(p[b, h, :len(o)], p0[b, h, o])
            assert torch.equal(w[b, h, :len(o)].nan_to_num(-7), w0[b, h, o].nan_to_num(-7))
            assert (w[b, h, len(o):budget] == 0).all() and (p[b, h, len(o):budget] == -1).all()
            if len(o):
                page, offset = pool.places(b, o)
                to_page, to_offset = pool.places(b, torch.arange(len(o), device=DEV))
                for new, old in ((pool.keys, keys), (pool.values, values)):
                    assert torch.equal(new[to_page, h, to_offset], old[page, h, offset])
                    old[to_page, h, to_offset] = new[to_page, h, to_offset]
    # nothing else was written
    assert torch.equal(keys.view(torch.int16), pool.keys.view(torch.int16)) and torch.equal(values.view(torch.int16), pool.values.view(torch.int16))


def eviction_state(lengths, heads, columns, seed, ties=0.3):
    g = torch.Generator(device=DEV).manual_seed(seed)
    weights = torch.exp(2 * torch.randn((len(lengths), heads, columns), generator=g, device=DEV))
    weights[torch.rand(weights.shape, generator=g, device=DEV) < ties] = 0.0
    seen = [2 * max(n, 0) + 3 for n in lengths]
    positions = torch.zeros((len(lengths), heads, columns), dtype=torch.int32, device=DEV)
    for b, n in enumerate(lengths):
        for h in range(heads):
            if n > 0:
                positions[b, h, :n] = torch.randperm(seen[b], generator=g, device=DEV)[:n]
    return weights, positions, seen


@pytest.mark.parametrize("lengths,budget,sink,recent", [
    ([300], 256, 4, 32), ([5000, 17, 0, -1, 257, 256], 256, 4, 100), ([3], 2, 0, 0), ([2], 1, 1, 0), ([1000, 900], 700, 0, 700),
    ([9000], 8192, 4, 512), ([20000, 4], 37, 3, 30), ([33], 32, 16, 16)])
@pytest.mark.parametrize("page,in_place", [(16, False), (24, True)])
def test_tokens_of_least_weight_leave(lengths, budget, sink, recent, page, in_place):
    pool = Pool(lengths, 2, 128, page, torch.bfloat16, seed=11)
    width = max(pool.columns * page, budget)
    weights, positions, seen = eviction_state(lengths, 2, width, 12)
    check_evict(pool, 2, lengths, seen, weights, positions, budget, sink, recent, in_place)


@pytest.mark.parametrize("heads,dim,dtype", [(1, 64, torch.float16), (8, 128, torch.float16)])
def test_eviction_of_other_shapes(heads, dim, dtype):
    lengths = [700, 64, 4100]
    pool = Pool(lengths, heads, dim, 32, dtype, seed=13)
    weights, positions, seen = eviction_state(lengths, heads, pool.columns * 32, 14)
    check_evict(pool, heads, lengths, seen, weights, positions, 512, 4, 64)


@pytest.mark.parametrize("budget", [1, 96, 500, 600])
@pytest.mark.parametrize("page,in_place", [(16, False), (24, "state"), (64, True)])
def test_eviction_of_many_short_rows(budget, page, in_place):
    lengths = [[1200, 0, 97, 513, -1, budget, budget + 1, 1100 + i][i % 8] for i in range(40)]
    pool = Pool(lengths, 8, 64, page, torch.float16, seed=23)
    weights, positions, seen = eviction_state(lengths, 8, pool.columns * page, 24)
    check_evict(pool, 8, lengths, seen, weights, positions, budget, 0, 1, in_place)


@pytest.mark.parametrize("value", [0.0, 1.5, -2.0, float("nan"), float("inf"), 1e-42])
def test_weights_that_all_tie(value):
    lengths = [1500]
    pool = Pool(lengths, 2, 128, 16, torch.bfloat16, seed=15)
    weights, positions, seen = eviction_state(lengths, 2, pool.columns * 16, 16)
    weights[:] = value
    check_evict(pool, 2, lengths, seen, weights, positions, 1000, 4, 50)


def test_order_of_special_weights():
    lengths = [700]
    pool = Pool(lengths, 1, 128, 16, torch.bfloat16, seed=17)
    weights, positions, seen = eviction_state(lengths, 1, pool.columns * 16, 18)
    specials = torch.tensor([float("nan"), float("-inf"), -3.0, -0.0, 0.0, 1e-42, -1e-42, 1.0, float("inf")], device=DEV)
    weights[0, 0, :700] = specials[torch.arange(700, device=DEV) % 9]
    for budget in (60, 200, 350, 500, 640, 699):
        check_evict(pool, 1, lengths, seen, weights, positions, budget, 0, 0)


def test_more_protected_tokens_than_the_budget_holds():
    """Positions are distinct in earnest; equal ones must not lead anywhere else than to the first places."""
    lengths = [600]
    pool = Pool(lengths, 2, 128, 16, torch.bfloat16, seed=19)
    weights, positions, seen = eviction_state(lengths, 2, pool.columns * 16, 20)
    positions[:] = 0
    check_evict(pool, 2, lengths, seen, weights, positions, 512, 4, 64)


def test_eviction_out_of_range():
    from inquant import _native as N
    from inquant.dense_paged import evict_tokens
    lengths = [600, 300]
    pool = Pool(lengths, 2, 128, 16, torch.bfloat16, seed=21)
    weights, positions, seen = eviction_state(lengths, 2, pool.columns * 16, 22)
    table = pool.table.clone()
    table[0, 30:] = 10 ** 9
    assert N.take_status(pool.keys.device) == 0
    kept = pool.keys.clone()
    n, w, p = evict_tokens(pool.keys, pool.values, table, pool.n, weights, positions, ints(seen), 256, sink=4, recent=64)
    assert N.take_status(pool.keys.device) == N.STATUS_BAD_INDEX and n.tolist() == [256, 256]
    other = torch.ones(pool.keys.shape[0], dtype=torch.bool, device=DEV)
    other[pool.table[0].long()] = False
    other[pool.table[1].long().clamp_min(0)] = False
    assert torch.equal(kept[other].view(torch.int16), pool.keys[other].view(torch.int16))
    n, _, _ = evict_tokens(pool.keys, pool.values, pool.table, ints([2 ** 31 - 1, 300]), weights, positions, ints(seen), 256)
    assert N.take_status(pool.keys.device) == N.STATUS_BAD_INDEX and n.tolist() == [256, 256]


@pytest.mark.parametrize("heads,q_heads,dim", [(2, 4, 128), (1, 20, 64)])
@pytest.mark.parametrize("page", [16, 24])
def test_a_new_token_whose_page_is_not_there_is_left_out(heads, q_heads, dim, page):
    """It is not stored, so that nothing attends to it and no weight is kept up for it."""
    from inquant import _native as N
    from inquant.dense_paged import paged_attention
    lengths = [12 * page, 12 * page + 5, 40, 0]
    pool = Pool(lengths, heads, dim, page, torch.bfloat16, seed=31)
    q, new_k, new_v = (query(4, h, dim, torch.bfloat16, s) for h, s in ((q_heads, 7), (heads, 8), (heads, 9)))
    old = torch.rand((4, heads, pool.columns * page), device=DEV)
    assert N.take_status(q.device) == 0
    for bad in (-1, pool.keys.shape[0], 2 ** 31 - 1):
        table = pool.table.clone()
        table[0, 12] = table[1, 12] = table[3, 0] = bad         # tokens 12 page ..: the new one alone, five and the new one, the new one alone
        kept = pool.keys.clone(), pool.values.clone()
        into = torch.full_like(old, 5.0)
        out, w = paged_attention(q, pool.keys, pool.values, table, pool.n, new_key=new_k, new_value=new_v, weights=old, out_weights=into)
        assert N.take_status(q.device) == N.STATUS_BAD_INDEX
        check_token(pool, q, out, tokens=[12 * page, 12 * page, 41, 0])
        for b, n in ((0, 12 * page), (1, 12 * page)):
            alone = paged_attention(q, pool.keys, pool.values, pool.table, ints([n if i == b else 0 for i in range(4)]),
                                    weights=old, out_weights=torch.zeros_like(old))[1]
            assert ((w[b, :, :n] - alone[b, :, :n]).abs() <= 2.0 ** -18 * w[b, :, :n]).all()
            assert (w[b, :, lengths[b]] == 0).all() and (w[b, :, lengths[b] + 1:] == 5).all()
        assert torch.equal(w[1, :, 12 * page:12 * page + 5], old[1, :, 12 * page:12 * page + 5])
        assert (w[3, :, 0] == 0).all()
        # request 2 has its page: its token was stored, and nothing else
        p, o = pool.places(2, torch.tensor([40], device=DEV))
        for now, before, new in zip((pool.keys, pool.values), kept, (new_k, new_v)):
            assert torch.equal(now[p, :, o][0], new[2])
            before[p, :, o] = new[2]
            assert torch.equal(now.view(torch.int16), before.view(torch.int16))


@pytest.mark.parametrize("lengths", [[1], [37, 200], [9000, 5, 0], [300] * 40])
@pytest.mark.parametrize("weights", [False, True])
def test_logits_that_are_all_minus_infinity_are_not_a_number(lengths, weights):
    """Zero divided by zero, as the formula has it and packed prompts give it; a row of the same request with one finite
    logit has that token, and a request without tokens zeros."""
    from inquant.dense_paged import paged_attention
    pool = Pool(lengths, 2, 128, 16, torch.bfloat16, seed=33, spare=1)
    q = query(len(lengths), 8, 128, torch.bfloat16)
    q[:, :, 0] = 1.0
    for b, n in enumerate(lengths):
        if n:
            p, o = pool.places(b, torch.arange(n, device=DEV))
            pool.keys[p, :, o, 0] = -math.inf
            p, o = pool.places(b, torch.tensor([n // 2], device=DEV))
            pool.keys[p, 1, o, 0] = 0.25     # the one token that heads 4 to 7 have
    into = torch.zeros((len(lengths), 2, pool.columns * 16), device=DEV) if weights else None
    got = paged_attention(q, pool.keys, pool.values, pool.table, pool.n, out_weights=into)
    out = got[0] if weights else got
    for b, n in enumerate(lengths):
        if n == 0:
            assert (out[b] == 0).all()
            continue
        p, o = pool.places(b, torch.tensor([n // 2], device=DEV))
        assert torch.isnan(out[b, :4]).all() and torch.equal(out[b, 4:], pool.values[p, 1, o].expand(4, 128))
        if weights:
            one = torch.zeros(n, device=DEV)
            one[n // 2] = 4.0
            assert torch.isnan(got[1][b, 0, :n]).all() and torch.equal(got[1][b, 1, :n], one)


def test_results_whose_rows_share_memory_are_refused_before_any_launch():
    """As without a GPU, where the native side of a call looks first."""
    from inquant.dense_paged import evict_tokens, paged_attention
    from inquant.prompt import prompt_attention, prompt_weights
    lengths = [300, 40]
    pool = Pool(lengths, 2, 128, 16, torch.bfloat16, seed=45)
    kept, q, width = pool.keys.clone(), query(2, 4, 128, torch.bfloat16), pool.columns * 16
    weights, positions, seen = eviction_state(lengths, 2, width, 46)
    decode, cut = (pool.keys, pool.values, pool.table, pool.n), (pool.keys, pool.values, pool.table, pool.n, weights, positions, ints(seen), 64)
    floats, whole = torch.zeros((1, 1, width), device=DEV), torch.zeros((1, 1, width), dtype=torch.int32, device=DEV)
    rows, cu = query(8, 4, 128, torch.bfloat16), ints([0, 8])
    for call in (lambda: paged_attention(q, *decode, out=q[:, :1].clone().expand(2, 4, 128)), lambda: paged_attention(q, *decode, out_weights=floats.expand(2, 2, width)),
                 lambda: paged_attention(q, *decode, weights=floats.expand(2, 2, width)), lambda: evict_tokens(*cut, sink=1, recent=2, out_weights=floats.expand(2, 2, width)),
                 lambda: evict_tokens(*cut, sink=1, recent=2, out_positions=whole.expand(2, 2, width)),
                 lambda: prompt_attention(rows, rows, rows, cu, out=torch.zeros(4096, dtype=rows.dtype, device=DEV).as_strided((8, 4, 128), (64, 128, 1))),
                 lambda: prompt_attention(rows, rows, rows, cu, lse=floats[0, :, :8].expand(4, 8)),
                 lambda: prompt_weights(rows, rows, torch.zeros((4, 8), device=DEV), cu, out=floats[0, :, :8].expand(4, 8))):
        with pytest.raises(ValueError):
            call()
    assert torch.equal(kept.view(torch.int16), pool.keys.view(torch.int16)) and (floats == 0).all() and (whole == 0).all()
    # what is only read may be the same row for all
    a = paged_attention(q, *decode, weights=floats.expand(2, 2, width), out_weights=torch.zeros((2, 2, width), device=DEV))
    b = paged_attention(q, *decode, out_weights=torch.zeros((2, 2, width), device=DEV))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# slices of a row per CTA of 2561 to 4608 tokens, of up to 8192 and of more, in one CTA per row and in clusters
@pytest.mark.parametrize("lengths,heads,budget", [
    ([4000, 2561, 100] + [3900] * 37, 8, 3000), ([7000, 4609, 8192] + [6000] * 37, 8, 5000), ([9000, 16385, 8193] + [9000 + i for i in range(37)], 8, 8500),
    ([70001], 2, 30000), ([131072, 50000], 1, 100000)])
@pytest.mark.parametrize("in_place", [False, "state", True])
def test_long_slices_of_rows(lengths, heads, budget, in_place):
    """Ties everywhere, across the borders of slices and of what a CTA looks at in one go."""
    pool = Pool(lengths, heads, 64, 64, torch.float16, seed=35)
    weights, positions, seen = eviction_state(lengths, heads, pool.columns * 64, 36, ties=0.7)
    check_evict(pool, heads, lengths, seen, weights, positions, budget, 4, 100, in_place)


def test_offsets_that_pass_32_bits_for_keys_and_values():
    """Pages that start between 2^31 and 5 2^30 elements: read, stored into and moved within."""
    from inquant.dense_paged import evict_tokens, paged_attention
    lengths, page_stride = [60], 2 ** 30
    pool = Pool(lengths, 2, 128, 16, torch.bfloat16, seed=37)
    q, new_k, new_v = (query(1, h, 128, torch.bfloat16, s) for h, s in ((14, 7), (2, 8), (2, 9)))
    table = ints([[5, 2, 4, 3]])
    assert pool.table.shape == table.shape and all(p * page_stride >= 2 ** 31 for p in table[0].tolist()) and 5 * page_stride > 2 ** 32
    keys, values = (torch.empty(5 * page_stride + 4096, dtype=torch.bfloat16, device=DEV).as_strided((6, 2, 16, 128), (page_stride, 2048, 128, 1)) for _ in range(2))
    keys[table[0].long()], values[table[0].long()] = pool.keys[pool.table[0].long()], pool.values[pool.table[0].long()]
    near, far = (pool.keys, pool.values, pool.table), (keys, values, table)
    old = torch.rand((1, 2, 64), device=DEV)
    steps = [paged_attention(q, *at, pool.n, new_key=new_k, new_value=new_v, weights=old, out_weights=torch.zeros_like(old)) for at in (near, far)]
    assert all(torch.equal(a, b) for a, b in zip(*steps))
    check_token(pool, q, steps[1][0], steps[1][1], old, fresh=True)
    positions = torch.arange(64, dtype=torch.int32, device=DEV).expand(1, 2, 64).contiguous()
    cuts = [evict_tokens(*at, ints([61]), steps[0][1], positions, ints([61]), 33, sink=2, recent=9) for at in (near, far)]
    assert all(torch.equal(a, b) for a, b in zip(*cuts))
    for there, here in ((keys, pool.keys), (values, pool.values)):
        a, b = there[table[0].long()], here[pool.table[0].long()]
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))


def ragged(count, longest, seed):
    g = torch.Generator().manual_seed(seed)
    return [[0, -1, 1, longest][b] if b < 4 else int(torch.randint(1, longest + 1, (1,), generator=g)) for b in range(count)]


def test_ranges_of_two_sizes():
    """More than 48 units of 64 tokens for each CTA: three quarters of an even share first, then eighths."""
    from inquant.dense_paged import paged_attention
    lengths = ragged(64, 8192, 38)
    pool = Pool(lengths, 8, 128, 16, torch.bfloat16, seed=39, spare=1)
    ctas = 2 * torch.cuda.get_device_properties(0).multi_processor_count
    assert sum(-(-max(n, 0) // 64) for n in lengths) * 8 > 48 * ctas
    q = query(64, 32, 128, torch.bfloat16)
    new_k, new_v = query(64, 8, 128, torch.bfloat16, 8), query(64, 8, 128, torch.bfloat16, 9)
    old = torch.rand((64, 8, pool.columns * 16), device=DEV)
    out, w = paged_attention(q, pool.keys, pool.values, pool.table, pool.n, new_key=new_k, new_value=new_v, weights=old, out_weights=torch.zeros_like(old))
    check_token(pool, q, out, w, old, fresh=True)


def test_a_captured_step_whose_ranges_change_their_kind():
    """One launch serves lengths that are cut evenly and lengths that are cut into ranges of two sizes."""
    from inquant.dense_paged import paged_attention
    mixes = [ragged(64, 8192, 40), [40] * 64, ragged(64, 8192, 41)[::-1], [0] * 63 + [8000], ragged(64, 5200, 42)]
    pool = Pool([8192] * 64, 8, 64, 64, torch.float16, seed=43)
    q = query(64, 32, 64, torch.float16)
    n, into = ints(mixes[0]), torch.zeros((64, 8, pool.columns * 64), device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = paged_attention(q, pool.keys, pool.values, pool.table, n, out_weights=into)
    for mix in mixes:
        n.copy_(ints(mix))
        graph.replay()
        check_token(pool, q, out, into, tokens=[max(x, 0) for x in mix])


@pytest.mark.parametrize("budget", [64, 300])
def test_a_captured_eviction_follows_lengths_and_weights(budget):
    from inquant.dense_paged import evict_tokens
    mixes = [[700, 64, 300], [301, 65, 1], [0, -1, 640]]
    pool = Pool([700] * 3, 2, 64, 16, torch.float16, seed=47)
    rows = pool.keys.clone(), pool.values.clone()
    states = [eviction_state(mix, 2, pool.columns * 16, 48 + i) for i, mix in enumerate(mixes)]
    weights, positions, n, seen = states[0][0].clone(), states[0][1].clone(), ints(mixes[0]), ints(states[0][2])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = evict_tokens(pool.keys, pool.values, pool.table, n, weights, positions, seen, budget, sink=2, recent=20)
    for mix, (w, p, s) in zip(mixes[::-1], states[::-1]):
        want_keys, want_values = rows[0].clone(), rows[1].clone()
        want = evict_tokens(want_keys, want_values, pool.table, ints(mix), w, p, ints(s), budget, sink=2, recent=20)
        pool.keys.copy_(rows[0]), pool.values.copy_(rows[1]), weights.copy_(w), positions.copy_(p), n.copy_(ints(mix)), seen.copy_(ints(s))
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert torch.equal(pool.keys.view(torch.int16), want_keys.view(torch.int16)) and torch.equal(pool.values.view(torch.int16), want_values.view(torch.int16))


def test_two_streams_at_once():
    """Decode and eviction of two caches, each on a stream of its own, over and over."""
    from inquant.dense_paged import evict_tokens, paged_attention
    pools = [Pool([4000, 900], 4, 128, 16, torch.bfloat16, seed=s) for s in (50, 51)]
    q = query(2, 28, 128, torch.bfloat16)
    width = pools[0].columns * 16
    states = [eviction_state([4000, 900], 4, width, s) for s in (52, 53)]

    def step(pool, state):
        keys, values = pool.keys.clone(), pool.values.clone()
        out, w = paged_attention(q, keys, values, pool.table, pool.n, weights=state[0], out_weights=torch.zeros_like(state[0]))
        left = evict_tokens(keys, values, pool.table, pool.n, w, state[1], ints(state[2]), 700, sink=4, recent=64)
        return out, w, *left, keys.view(torch.int16), values.view(torch.int16)

    want = [step(*both) for both in zip(pools, states)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in pools], [[], []]
    for _ in range(8):
        for i, both in enumerate(zip(pools, states)):
            with torch.cuda.stream(streams[i]):
                got[i].append(step(*both))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for each in got[i] for a, b in zip(each, want[i]))
