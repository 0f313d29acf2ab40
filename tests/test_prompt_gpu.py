"""Packed prompts (``inquant.prompt``) against their formulas in 64 bits.

Bounds.  u is half a step of the dtype.  A logit's fp32 error is at most delta = D 2^-24 scale sum |q_c k_c| (D sums of exact
products), which is the relative error of its exponential; 2^-20 covers the exponential unit and fp32 sums of up
to a few thousand addends in chains of 128 and less.  A probability is rounded to the dtype once (u) before the product
with the values, its normaliser is not (2 delta for both), and the result is rounded once (u):
|out - exact| <= sum p |v| (u + 2 delta + 2^-20) + u |exact| (1 + u)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def starts(lengths):
    return [sum(lengths[:i]) for i in range(len(lengths) + 1)]


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def states(lengths, keys, q_heads, heads, dim, dtype, seed=0, behind=0, spread=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    q, k, v = (torch.randn((n + behind, h, dim), generator=g, device=DEV) * s
               for n, h, s in ((sum(lengths), q_heads, spread), (sum(keys), heads, spread), (sum(keys), heads, 1.0)))
    return q.to(dtype), k.to(dtype), v.to(dtype)


def formula(q, k, v, lengths, keys, scale, window=0):
    """Output, its bound, log-sum-exp and its bound, weights and their bound, per packed row, in 64 bits."""
    q, k, v = q.double(), k.double(), v.double()
    dim, group, u = q.shape[2], q.shape[1] // k.shape[1], None
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    lse = torch.full((q.shape[1], q.shape[0]), -math.inf, dtype=torch.float64, device=q.device)
    lse_bound = torch.zeros_like(lse)
    weights = torch.zeros((k.shape[1], k.shape[0]), dtype=torch.float64, device=q.device)
    w_bound = torch.zeros_like(weights)
    qs, ks = starts(lengths), starts(keys)
    for b, (n, m) in enumerate(zip(lengths, keys)):
        rows, cols = slice(qs[b], qs[b] + n), slice(ks[b], ks[b] + m)
        if not n or not m:
            continue
        sees = torch.arange(m, device=q.device) <= (m - n) + torch.arange(n, device=q.device)[:, None]
        some = sees.any(1)
        for h in range(q.shape[1]):
            kh, vh = k[cols, h // group], v[cols, h // group]
            logits = (q[rows, h] @ kh.T * scale).masked_fill(~sees, -math.inf)
            delta = dim * 2.0 ** -24 * scale * (q[rows, h].abs() @ kh.abs().T).masked_fill(~sees, 0).amax(1) + 2.0 ** -20
            sums = torch.logsumexp(logits, 1)
            p = torch.where(some[:, None], torch.exp(logits - torch.where(some, sums, 0.0)[:, None]), 0.0)
            out[rows, h] = p @ torch.where(sees.any(0)[:, None], vh, 0.0)
            bound[rows, h] = p @ torch.where(sees.any(0)[:, None], vh.abs(), 0.0)
            bound[rows, h] = torch.complex(bound[rows, h], torch.zeros_like(bound[rows, h])).real
            lse[h, rows] = sums
            lse_bound[h, rows] = delta + 2.0 ** -22 * torch.where(some, sums.abs(), 0.0)
            counted = torch.arange(n, device=q.device) >= (n - window if window else 0)
            weights[h // group, cols] += p[counted].sum(0)
            w_bound[h // group, cols] += (p * (2 * delta[:, None] + 2.0 ** -21 * torch.where(some, sums.abs(), 0.0)[:, None]))[counted].sum(0)
    delta_out = lse_bound.T.unsqueeze(-1)
    return out, bound, delta_out, lse, lse_bound, weights, w_bound


def check(q, k, v, lengths, keys, scale=None, window=0, cu_offset=0):
    from inquant import _native as N
    from inquant.prompt import prompt_attention, prompt_weights
    scale = q.shape[2] ** -0.5 if scale is None else scale
    cu, cu_k = ints(starts(lengths)), ints(starts(keys))
    out, lse = prompt_attention(q, k, v, cu, cu_k, scale=scale)
    w = prompt_weights(q, k, lse, cu, cu_k, scale=scale, window=window or None)
    assert N.take_status(q.device) == 0      # no wait gave up
    want, share, delta, want_lse, lse_bound, want_w, w_bound = formula(q, k, v, lengths, keys, scale, window)
    n, m, u = sum(lengths), sum(keys), unit(q.dtype)
    off = (out[:n].double() - want[:n]).abs()
    allowed = share[:n] * (u + 2 * delta[:n]) + u * want[:n].abs() * (1 + u) + torch.finfo(q.dtype).smallest_normal
    assert (off <= allowed).all(), (off / allowed).max()
    same = torch.isinf(want_lse[:, :n])
    assert torch.equal(torch.isinf(lse[:, :n]) & (lse[:, :n] < 0), same)
    assert ((lse[:, :n].double() - want_lse[:, :n]).abs() <= lse_bound[:, :n])[~same].all()
    assert ((w[:, :m].double() - want_w[:, :m]).abs() <= w_bound[:, :m] + 1e-30).all()
    return out, lse, w


SHAPES = [(28, 4, 128, torch.bfloat16), (8, 8, 128, torch.float16), (32, 2, 64, torch.float16), (5, 1, 64, torch.bfloat16)]


@pytest.mark.parametrize("q_heads,heads,dim,dtype", SHAPES)
@pytest.mark.parametrize("lengths", [[1], [2], [127], [128], [129], [255], [256], [257], [513], [1100]])
def test_one_prompt_of_any_length(q_heads, heads, dim, dtype, lengths):
    q, k, v = states(lengths, lengths, q_heads, heads, dim, dtype, spread=1.5)
    check(q, k, v, lengths, lengths)


@pytest.mark.parametrize("q_heads,heads,dim,dtype", SHAPES)
@pytest.mark.parametrize("lengths,past", [([3, 0, 300, 1, 257, 64], [0] * 6), ([5, 130, 1, 40], [700, 3, 129, 0]),
                                          ([1] * 70, list(range(70))), ([17] * 33 + [400], [0] * 34), ([0, 0, 9], [0, 50, 0]),
                                          ([3] * 150 + [0, 300] + [1] * 150, [0] * 100 + [20] * 202)])
@pytest.mark.parametrize("window", [0, 1, 33])
def test_packed_prompts_behind_histories(q_heads, heads, dim, dtype, lengths, past, window):
    keys = [n + p for n, p in zip(lengths, past)]
    q, k, v = states(lengths, keys, q_heads, heads, dim, dtype, seed=1)
    check(q, k, v, lengths, keys, window=window)


@pytest.mark.parametrize("lengths,keys", [([9], [4]), ([300, 5], [20, 0]), ([600, 2], [290, 3]), ([4], [0])])
def test_queries_without_a_key_give_zeros(lengths, keys):
    q, k, v = states(lengths, keys, 8, 2, 128, torch.bfloat16)
    out, lse, _ = check(q, k, v, lengths, keys)
    blind = lengths[0] - keys[0]
    assert (out[:blind] == 0).all() and torch.isneginf(lse[:, :blind]).all()


@pytest.mark.parametrize("dim,dtype", [(128, torch.bfloat16), (64, torch.float16)])
@pytest.mark.parametrize("lengths,keys", [([256], [9000]), ([40, 3], [5000, 6200])])
def test_long_histories_are_cut_and_joined(dim, dtype, lengths, keys):
    """Few rows over many keys: the items are cut into segments."""
    from inquant import _native as N
    q, k, v = states(lengths, keys, 4, 2, dim, dtype, seed=3)
    assert N.library().inq_prompt_workspace_bytes(4, 2, dim, q.shape[0], k.shape[0], len(lengths), 0, 0) > 0
    check(q, k, v, lengths, keys)


def test_long_prompt_of_many_steps_per_item():
    q, k, v = states([2900], [2900], 7, 1, 128, torch.bfloat16, seed=4)
    check(q, k, v, [2900], [2900], window=1000)


@pytest.mark.parametrize("dim,dtype", [(128, torch.bfloat16), (64, torch.float16)])
@pytest.mark.parametrize("lengths,past", [([17, 900, 256, 1, 1300, 640, 90, 128, 1100, 333, 512, 700], [0] * 12), ([130, 0, 300, 60, 500], [1900, 700, 40, 2500, 1000])])
def test_many_items_per_sm(lengths, past, dim, dtype):
    """Items with and without a second tile, of one step to many, one behind the other in a CTA."""
    keys = [n + p for n, p in zip(lengths, past)]
    q, k, v = states(lengths, keys, 32, 8, dim, dtype, seed=11)
    check(q, k, v, lengths, keys)


def test_large_logits_raise_the_reference_maximum():
    q, k, v = states([900], [900], 4, 2, 128, torch.bfloat16, seed=5)
    k *= torch.linspace(0.1, 6, 900, device=DEV)[:, None, None].to(k.dtype)      # later keys have ever larger logits
    check(q, k, v, [900], [900])


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_what_a_query_does_not_see_does_not_reach_it(dim, value):
    """Non-finite values behind a sequence and at later positions; rows that see them have them."""
    from inquant.prompt import prompt_attention
    lengths = [150, 300, 70]
    q, k, v = states(lengths, lengths, 4, 2, dim, torch.bfloat16, seed=6, behind=60)
    cu = ints(starts(lengths))
    clean_out, clean_lse = prompt_attention(q, k, v, cu)
    k2, v2, q2 = k.clone(), v.clone(), q.clone()
    at = [150 + 200, 150 + 299, 150 + 40]        # positions 200, 299 and 40 of the second sequence
    v2[at[0], 1, 5] = value
    v2[at[1], 0] = value
    k2[520:], v2[520:], q2[520:] = value, value, value       # behind the last sequence
    out, lse = prompt_attention(q2, k2, v2, cu)
    assert torch.equal(lse[:, :520], clean_lse[:, :520])
    group = 2
    seen = torch.zeros_like(clean_out, dtype=torch.bool)
    seen[150 + 200:450, group:, 5] = True
    seen[449, :group] = True
    seen = seen[:520]
    assert torch.equal(out[:520][~seen], clean_out[:520][~seen])
    got = out[:520][seen].float()
    assert (torch.isnan(got) if math.isnan(value) else got == value).all()
    k2[at[2]] = float("nan")                      # a key that is not a number: nothing before it changes
    out, lse = prompt_attention(q2, k2, v2, cu)
    before = torch.cat([torch.arange(150 + 40), torch.arange(450, 520)]).to(DEV)
    assert torch.equal(out[before], clean_out[before]) and torch.isnan(out[150 + 40:150 + 200]).all()


def test_infinities_of_both_signs_are_not_a_number():
    from inquant.prompt import prompt_attention
    q, k, v = states([100], [100], 2, 1, 128, torch.float16)
    v[10, 0, 3], v[20, 0, 3] = float("inf"), float("-inf")
    out, _ = prompt_attention(q, k, v, ints([0, 100]))
    column = out[:, :, 3]
    assert torch.isfinite(column[:10]).all() and (column[10:20] == float("inf")).all() and torch.isnan(column[20:]).all()


def test_rows_of_no_sequence_stay_as_they_were():
    from inquant.prompt import prompt_attention, prompt_weights
    lengths = [40, 0, 300]
    q, k, v = states(lengths, lengths, 4, 2, 128, torch.bfloat16, behind=90)
    cu = ints([5 + s for s in starts(lengths)])
    out, lse = torch.full_like(q, 7), torch.full((4, q.shape[0]), 7.0, device=DEV)
    weights = torch.full((2, k.shape[0]), 7.0, device=DEV)
    prompt_attention(q, k, v, cu, out=out, lse=lse)
    prompt_weights(q, k, lse, cu, out=weights)
    for t in (out[:5], out[345:], lse[:, :5], lse[:, 345:], weights[:, :5], weights[:, 345:]):
        assert (t == 7).all()
    inner, inner_lse = prompt_attention(q[5:345].contiguous(), k[5:345].contiguous(), v[5:345].contiguous(), ints(starts(lengths)))
    assert torch.equal(out[5:345], inner) and torch.equal(lse[:, 5:345], inner_lse)


def test_strides_and_alignment():
    from inquant.prompt import prompt_attention, prompt_weights
    lengths = [200, 77]
    q, k, v = states(lengths, lengths, 8, 2, 128, torch.bfloat16, seed=8)
    cu = ints(starts(lengths))
    want, want_lse = prompt_attention(q, k, v, cu)
    want_w = prompt_weights(q, k, want_lse, cu)
    packed = torch.cat([q, k, v], 1)                               # a fused projection's output
    q2, k2, v2 = packed[:, :8], packed[:, 8:10], packed[:, 10:]
    head_major = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    shifted = [torch.empty(t.numel() + 3, dtype=t.dtype, device=DEV)[3:].view(t.shape).copy_(t) for t in (q, k, v)]
    reverse = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]      # channels are not neighbours
    for q3, k3, v3 in ((q2, k2, v2), head_major, shifted, reverse):
        room = torch.empty(277, 8, 256, dtype=q.dtype, device=DEV)[:, :, :128]
        out, lse = prompt_attention(q3, k3, v3, cu, out=room, lse=torch.empty(8, 300, device=DEV)[:, :277])
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
        assert torch.equal(prompt_weights(q3, k3, lse, cu), want_w)


def test_offsets_outside_the_tensors_are_cut_and_reported():
    from inquant import _native as N
    from inquant.prompt import prompt_attention, prompt_weights
    q, k, v = states([300], [300], 4, 2, 128, torch.bfloat16)
    want, want_lse = prompt_attention(q, k, v, ints([0, 300]))
    assert N.take_status(q.device) == 0
    for bad in ([0, 1000], [-7, 300], [-2147483648, 2147483647]):
        out, lse = prompt_attention(q, k, v, ints(bad))
        assert N.take_status(q.device) == N.STATUS_BAD_INDEX and torch.equal(out, want)
        prompt_weights(q, k, lse, ints(bad))
        assert N.take_status(q.device) == N.STATUS_BAD_INDEX
    prompt_attention(q, k, v, ints([0, 200, 100, 300]))
    assert N.take_status(q.device) == N.STATUS_BAD_INDEX


def test_captured_for_one_mix_of_lengths_and_replayed_for_another():
    from inquant.prompt import prompt_attention, prompt_weights
    q, k, v = states([400], [400], 8, 2, 128, torch.bfloat16)
    cu = ints([0, 100, 400])
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        prompt_attention(q, k, v, cu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out, lse = prompt_attention(q, k, v, cu)
        w = prompt_weights(q, k, lse, cu)
    for mix in ([0, 100, 400], [0, 399, 400], [0, 0, 400]):
        cu.copy_(ints(mix))
        graph.replay()
        torch.cuda.synchronize()
        want, want_lse = prompt_attention(q, k, v, ints(mix))
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
        assert torch.equal(w, prompt_weights(q, k, want_lse, ints(mix)))


def test_two_streams_at_once():
    from inquant.prompt import prompt_attention
    cases = [states([256], [4000], 4, 2, 128, torch.bfloat16, seed=s) for s in (1, 2)]
    cu, cu_k = ints([0, 256]), ints([0, 4000])
    want = [prompt_attention(*c, cu, cu_k) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(5):
        for i, c in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                got[i].append(prompt_attention(*c, cu, cu_k))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i][0]) and torch.equal(l, want[i][1]) for o, l in got[i])


def test_agrees_with_the_attention_of_one_sequence():
    from inquant.prefill import prefill_attention
    from inquant.prompt import prompt_attention
    q, k, v = states([700], [1500], 28, 4, 128, torch.bfloat16, seed=9)
    single = prefill_attention(*(t.transpose(0, 1).unsqueeze(0) for t in (q, k, v)))[0].transpose(0, 1)
    out, _ = prompt_attention(q, k, v, ints([0, 700]), ints([0, 1500]))
    assert (out.float() - single.float()).abs().max() <= 2 * unit(q.dtype) * v.abs().max().float()


@pytest.mark.parametrize("dim,dtype", [(128, torch.bfloat16), (64, torch.float16)])
@pytest.mark.parametrize("lengths", [[100, 300, 128, 260, 17, 290, 129, 200] * 7, [60, 1100, 90, 500, 256, 30] * 5])
def test_values_that_are_not_finite_stay_with_the_rows_that_see_them(dim, dtype, lengths):
    """Many items behind one another in a CTA, with and without a second tile, some with values that are not finite: what one
    item found is neither lost to its own rows nor handed to those of another."""
    from inquant.prompt import prompt_attention
    heads, q_heads = 8, 32
    q, k, v = states(lengths, lengths, q_heads, heads, dim, dtype, seed=21)
    clean, clean_lse, _ = check(q, k, v, lengths, lengths)
    first = starts(lengths)
    cu = ints(first)
    specials = torch.tensor([math.inf, -math.inf, math.nan])
    where = torch.zeros(sum(lengths), dtype=torch.long, device=DEV)       # first row of the row's sequence
    for b, n in enumerate(lengths):
        where[first[b]:first[b] + n] = first[b]
    row = torch.arange(sum(lengths), device=DEV)
    g = torch.Generator().manual_seed(22)
    for turn in range(6):
        values = v.clone()
        kinds = [torch.zeros(v.shape, dtype=torch.bool, device=DEV) for _ in specials]
        for b, n in enumerate(lengths):
            if (b + turn) % 3 == 0:
                continue        # nothing to find between two that have something
            for _ in range(4):
                at, h, c, kind = (int(torch.randint(m, (1,), generator=g)) for m in (n, heads, dim, 3))
                values[first[b] + at, h, c] = specials[kind]
                for i in range(3):
                    kinds[i][first[b] + at, h, c] = i == kind
        seen = []
        for kind in kinds:      # whether a row's sequence has one at or before the row
            total = torch.cat([torch.zeros_like(kind[:1], dtype=torch.int32), kind.to(torch.int32).cumsum(0, dtype=torch.int32)])
            seen.append((total[row + 1] > total[where]).repeat_interleave(q_heads // heads, 1))
        plus, minus, nan = seen
        want = torch.where(plus, math.inf, clean.float())
        want = torch.where(minus, -math.inf, want)
        want = torch.where(nan | (plus & minus), math.nan, want)
        # a channel's result depends on that channel's values alone: where a row sees nothing of the kind it is bit by bit what it was
        out, lse = prompt_attention(q, k, values, cu)
        assert torch.equal(out.float().nan_to_num(1e30), want.nan_to_num(1e30)), turn
        assert torch.equal(torch.isnan(out), torch.isnan(want)) and torch.equal(lse, clean_lse)
