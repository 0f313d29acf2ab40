"""What the calls over packed prompts and uncompressed pages refuse, and the bookkeeping of ``DensePagedCache`` (no GPU: every
refusal comes before the first launch)."""
import contextlib
import ctypes

import pytest
import torch

from inquant import _native as N

from inquant.dense_paged import DensePagedCache, evict_tokens, paged_attention
from inquant.prompt import prompt_attention, prompt_weights

BF16 = torch.bfloat16


@pytest.fixture
def no_device(monkeypatch):
    """CPU tensors pass for the device's, and a call that is not refused is noticed."""
    monkeypatch.setattr(N, "require_cuda", lambda *_: None)
    monkeypatch.setattr(N, "library", lambda: pytest.fail("not refused"))
    monkeypatch.setattr(N, "status_word", lambda _device: torch.zeros(1, dtype=torch.int32))


def offsets(*values):
    return torch.tensor(values, dtype=torch.int32)


def prompt_case(**changes):
    case = dict(query=torch.zeros(8, 4, 128, dtype=BF16), key=torch.zeros(8, 2, 128, dtype=BF16), value=torch.zeros(8, 2, 128, dtype=BF16),
                cu_seqlens=offsets(0, 3, 8))
    return {**case, **changes}


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="requires CUDA"):
        prompt_attention(**prompt_case())
    case = prompt_case()
    with pytest.raises(RuntimeError, match="requires CUDA"):
        prompt_weights(case["query"], case["key"], torch.zeros(4, 8), case["cu_seqlens"])
    with pytest.raises(RuntimeError, match="requires CUDA"):
        paged_attention(**paged_case())
    with pytest.raises(RuntimeError, match="requires CUDA"):
        evict_tokens(**evict_case())


@pytest.mark.parametrize("error,changes", [
    (ValueError, dict(query=torch.zeros(8, 512, dtype=BF16))),
    (ValueError, dict(key=torch.zeros(1, 8, 2, 128, dtype=BF16))),
    (ValueError, dict(value=torch.zeros(7, 2, 128, dtype=BF16))),
    (NotImplementedError, dict(query=torch.zeros(8, 4, 128))),
    (NotImplementedError, dict(value=torch.zeros(8, 2, 128, dtype=torch.float16))),
    (NotImplementedError, dict(query=torch.zeros(8, 4, 96, dtype=BF16), key=torch.zeros(8, 2, 96, dtype=BF16), value=torch.zeros(8, 2, 96, dtype=BF16))),
    (NotImplementedError, dict(key=torch.zeros(8, 2, 64, dtype=BF16), value=torch.zeros(8, 2, 64, dtype=BF16))),
    (ValueError, dict(query=torch.zeros(8, 5, 128, dtype=BF16))),
    (ValueError, dict(key=torch.zeros(8, 0, 128, dtype=BF16), value=torch.zeros(8, 0, 128, dtype=BF16))),
    (ValueError, dict(cu_seqlens=torch.tensor([0, 8]))),
    (ValueError, dict(cu_seqlens=offsets(0))),
    (ValueError, dict(cu_seqlens_k=offsets(0, 8))),
    (ValueError, dict(cu_seqlens_k=torch.tensor([0.0, 3, 8]))),
    (ValueError, dict(scale=0.0)), (ValueError, dict(scale=float("nan"))), (ValueError, dict(scale=-1)),
    (ValueError, dict(out=torch.zeros(8, 4, 128))), (ValueError, dict(out=torch.zeros(7, 4, 128, dtype=BF16))),
    (ValueError, dict(out=torch.zeros(8, 4, 132, dtype=BF16)[:, :, 4:])),
    (ValueError, dict(lse=torch.zeros(8, 4))), (ValueError, dict(lse=torch.zeros(8, 4).T)), (ValueError, dict(lse=torch.zeros(4, 8, dtype=BF16))),
])
def test_prompt_attention_refuses(no_device, error, changes):
    with pytest.raises(error):
        prompt_attention(**prompt_case(**changes))


@pytest.mark.parametrize("error,changes", [
    (ValueError, dict(lse=torch.zeros(8, 4))), (ValueError, dict(lse=torch.zeros(4, 8, dtype=BF16))), (ValueError, dict(window=0)),
    (ValueError, dict(window=-3)), (ValueError, dict(out=torch.zeros(2, 9))), (ValueError, dict(out=torch.zeros(2, 8, dtype=BF16))),
    (ValueError, dict(out=torch.zeros(8, 2).T)), (ValueError, dict(scale=0)), (ValueError, dict(cu_seqlens_k=offsets(0, 8))),
    (NotImplementedError, dict(key=torch.zeros(8, 2, 128))),
])
def test_prompt_weights_refuses(no_device, error, changes):
    case = prompt_case(lse=torch.zeros(4, 8))
    del case["value"]
    with pytest.raises(error):
        prompt_weights(**{**case, **changes})


def paged_case(**changes):
    case = dict(query=torch.zeros(3, 4, 128, dtype=BF16), key_pages=torch.zeros(5, 2, 16, 128, dtype=BF16),
                value_pages=torch.zeros(5, 2, 16, 128, dtype=BF16), block_table=torch.zeros(3, 2, dtype=torch.int32), lengths=offsets(1, 2, 3))
    return {**case, **changes}


@pytest.mark.parametrize("error,changes", [
    (ValueError, dict(query=torch.zeros(2, 4, 128, dtype=BF16))), (ValueError, dict(query=torch.zeros(3, 5, 128, dtype=BF16))),
    (ValueError, dict(query=torch.zeros(3, 4, 64, dtype=BF16))), (NotImplementedError, dict(query=torch.zeros(3, 4, 128, dtype=torch.float16))),
    (ValueError, dict(value_pages=torch.zeros(5, 2, 32, 128, dtype=BF16))), (ValueError, dict(key_pages=torch.zeros(5, 16, 128, dtype=BF16))),
    (NotImplementedError, dict(key_pages=torch.zeros(5, 2, 16, 128), value_pages=torch.zeros(5, 2, 16, 128))),
    (NotImplementedError, dict(key_pages=torch.zeros(5, 2, 16, 32, dtype=BF16), value_pages=torch.zeros(5, 2, 16, 32, dtype=BF16))),
    (ValueError, dict(key_pages=torch.zeros(5, 2, 128, 16, dtype=BF16).transpose(2, 3))),
    (ValueError, dict(value_pages=torch.zeros(5 * 2 * 16 * 128 + 1, dtype=BF16)[1:].view(5, 2, 16, 128))),
    (ValueError, dict(block_table=torch.zeros(3, 2, dtype=torch.int64))), (ValueError, dict(block_table=torch.zeros(3, 0, dtype=torch.int32))),
    (ValueError, dict(block_table=torch.zeros(2, 3, dtype=torch.int32).T)), (ValueError, dict(lengths=offsets(1, 2))),
    (ValueError, dict(lengths=torch.tensor([1, 2, 3]))), (ValueError, dict(new_key=torch.zeros(3, 2, 128, dtype=BF16))),
    (ValueError, dict(new_key=torch.zeros(3, 2, 128, dtype=BF16), new_value=torch.zeros(3, 1, 128, dtype=BF16))),
    (ValueError, dict(weights=torch.zeros(3, 2, 31))), (ValueError, dict(weights=torch.zeros(3, 1, 32))),
    (ValueError, dict(weights=torch.zeros(3, 2, 32, dtype=BF16))), (ValueError, dict(out_weights=torch.zeros(32, 2, 3).permute(2, 1, 0))),
    (ValueError, dict(out=torch.zeros(3, 4, 128))), (ValueError, dict(out=torch.zeros(3, 4, 129, dtype=BF16)[:, :, 1:])), (ValueError, dict(scale=0.0)),
])
def test_paged_attention_refuses(no_device, error, changes):
    with pytest.raises(error):
        paged_attention(**paged_case(**changes))


def evict_case(**changes):
    case = paged_case(weights=torch.zeros(3, 2, 32), positions=torch.zeros(3, 2, 32, dtype=torch.int32), seen=offsets(9, 9, 9), budget=8, sink=2, recent=3)
    del case["query"]
    return {**case, **changes}


@pytest.mark.parametrize("error,changes", [
    (ValueError, dict(budget=0)), (ValueError, dict(budget=4)), (ValueError, dict(sink=-1)), (ValueError, dict(recent=-1)), (ValueError, dict(budget=2 ** 31)),
    (ValueError, dict(seen=offsets(9, 9))), (ValueError, dict(seen=torch.tensor([9, 9, 9]))), (ValueError, dict(weights=torch.zeros(2, 2, 32))),
    (ValueError, dict(positions=torch.zeros(3, 2, 31, dtype=torch.int32))), (ValueError, dict(positions=torch.zeros(3, 2, 32))),
    (ValueError, dict(out_weights=torch.zeros(3, 2, 7))), (ValueError, dict(out_positions=torch.zeros(3, 2, 7, dtype=torch.int32))),
    (ValueError, dict(out_lengths=torch.zeros(3))), (ValueError, dict(out_lengths=torch.zeros(6, dtype=torch.int32)[::2])),
    (ValueError, dict(lengths=offsets(1))), (NotImplementedError, dict(key_pages=torch.zeros(5, 2, 16, 128), value_pages=torch.zeros(5, 2, 16, 128))),
])
def test_evict_tokens_refuses(no_device, error, changes):
    with pytest.raises(error):
        evict_tokens(**evict_case(**changes))


def test_empty_calls_launch_nothing(no_device):
    out, lse = prompt_attention(**prompt_case(query=torch.zeros(0, 4, 128, dtype=BF16)))
    assert out.shape == (0, 4, 128) and lse.shape == (4, 0)
    empty = torch.zeros(0, 2, 128, dtype=BF16)
    assert prompt_weights(torch.zeros(8, 4, 128, dtype=BF16), empty, torch.zeros(4, 8), offsets(0, 8), offsets(0, 0)).shape == (2, 0)
    none = dict(block_table=torch.zeros(0, 2, dtype=torch.int32), lengths=torch.zeros(0, dtype=torch.int32))
    assert paged_attention(**paged_case(query=torch.zeros(0, 4, 128, dtype=BF16), **none)).shape == (0, 4, 128)
    n, w, p = evict_tokens(**evict_case(weights=torch.zeros(0, 2, 32), positions=torch.zeros(0, 2, 32, dtype=torch.int32),
                                        seen=torch.zeros(0, dtype=torch.int32), **none))
    assert n.shape == (0,) and w.shape == (0, 2, 8) and p.shape == (0, 2, 8)


# ------------------------------------------------------------------------------------------------ C interface
def filled(kind):
    """Arguments that the entry point would take (addresses that nothing reads, because each test spoils one field)."""
    a, word, at = kind(), 4096, {}
    for name, ctype in kind._fields_:
        if ctype is ctypes.c_void_p:
            setattr(a, name, word)
    at.update({f: 128 for f, _ in kind._fields_ if "stride" in f})
    at.update(scale=1.0, head_dim=128, dtype=N.BF16, q_heads=4, kv_heads=2, n_seq=1, q_rows=3, k_rows=3, requests=2, pages=4, page_tokens=16,
              table_columns=2, budget=8, sink=1, recent=2, columns=32, workspace_bytes=1 << 40, window=0)
    for name, value in at.items():
        if name in {f for f, _ in kind._fields_}:
            setattr(a, name, value)
    return a


@pytest.mark.parametrize("function,kind,field,value,want", [
    (f, N.PromptArgs, *case) for f in ("inq_prompt_attention", "inq_prompt_weights") for case in [
        ("q", None, N.ERR_ARGUMENT), ("k", None, N.ERR_ARGUMENT), ("cu_q", None, N.ERR_ARGUMENT), ("cu_k", None, N.ERR_ARGUMENT),
        ("status", None, N.ERR_ARGUMENT), ("q_heads", 5, N.ERR_ARGUMENT), ("kv_heads", 0, N.ERR_ARGUMENT), ("n_seq", 0, N.ERR_ARGUMENT),
        ("q_rows", 0, N.ERR_ARGUMENT), ("k_rows", 1 << 31, N.ERR_CAPACITY), ("scale", 0.0, N.ERR_ARGUMENT), ("scale", float("nan"), N.ERR_ARGUMENT),
        ("dtype", N.F32, N.ERR_UNSUPPORTED), ("head_dim", 96, N.ERR_UNSUPPORTED), ("q", 4098, N.ERR_ARGUMENT), ("k_stride_t", 132, N.ERR_ARGUMENT),
        ("q_stride_h", -128, N.ERR_ARGUMENT)]
] + [("inq_prompt_attention", N.PromptArgs, "v", None, N.ERR_ARGUMENT), ("inq_prompt_attention", N.PromptArgs, "out", 4100, N.ERR_ARGUMENT),
     ("inq_prompt_attention", N.PromptArgs, "o_stride_t", 4, N.ERR_ARGUMENT), ("inq_prompt_weights", N.PromptArgs, "lse", None, N.ERR_ARGUMENT),
     ("inq_prompt_weights", N.PromptArgs, "weights", None, N.ERR_ARGUMENT), ("inq_prompt_weights", N.PromptArgs, "window", -1, N.ERR_ARGUMENT)]
    + [("inq_paged_attention", N.PagedAttentionArgs, *case) for case in [
        ("q", None, N.ERR_ARGUMENT), ("k", 4100, N.ERR_ARGUMENT), ("table", None, N.ERR_ARGUMENT), ("lengths", None, N.ERR_ARGUMENT),
        ("counters", None, N.ERR_ARGUMENT), ("status", None, N.ERR_ARGUMENT), ("new_k", None, N.ERR_ARGUMENT), ("out_weights", None, N.ERR_ARGUMENT),
        ("requests", 0, N.ERR_ARGUMENT), ("q_heads", 3, N.ERR_ARGUMENT), ("page_tokens", 0, N.ERR_ARGUMENT), ("table_columns", 0, N.ERR_ARGUMENT),
        ("pages", 0, N.ERR_ARGUMENT), ("scale", -1.0, N.ERR_ARGUMENT), ("dtype", N.F32, N.ERR_UNSUPPORTED), ("head_dim", 256, N.ERR_UNSUPPORTED),
        ("k_stride_t", 4, N.ERR_ARGUMENT), ("table_columns", 1 << 30, N.ERR_CAPACITY)]]
    + [("inq_evict_tokens", N.EvictArgs, *case) for case in [
        ("k", None, N.ERR_ARGUMENT), ("v", 4100, N.ERR_ARGUMENT), ("weights", None, N.ERR_ARGUMENT), ("positions", None, N.ERR_ARGUMENT),
        ("out_lengths", None, N.ERR_ARGUMENT), ("seen", None, N.ERR_ARGUMENT), ("budget", 0, N.ERR_ARGUMENT), ("budget", 2, N.ERR_ARGUMENT),
        ("sink", -1, N.ERR_ARGUMENT), ("recent", 1 << 30, N.ERR_ARGUMENT), ("head_dim", 12, N.ERR_UNSUPPORTED), ("v_stride_p", 4, N.ERR_ARGUMENT),
        ("table_columns", 1 << 20, N.ERR_CAPACITY), ("workspace", None, N.ERR_CAPACITY), ("workspace_bytes", 8, N.ERR_CAPACITY)]])
def test_entry_points_refuse_before_any_launch(function, kind, field, value, want):
    a = filled(kind)
    setattr(a, field, value)
    assert getattr(N.library(), function)(ctypes.byref(a), None) == want


def test_entry_points_refuse_no_arguments():
    for name in ("inq_prompt_attention", "inq_prompt_weights", "inq_paged_attention", "inq_evict_tokens"):
        assert getattr(N.library(), name)(None, None) == N.ERR_ARGUMENT


def test_structs_are_laid_out_as_the_header_says(tmp_path):
    import os
    import subprocess
    header = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "inquant_b200.h")
    kinds = [("inq_prompt_args_t", N.PromptArgs), ("inq_paged_attention_args_t", N.PagedAttentionArgs), ("inq_evict_args_t", N.EvictArgs)]
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{header}"', "int main(void) {"]
    want = []
    for name, kind in kinds:
        lines.append(f'  printf("%zu\\n", sizeof({name}));')
        want.append(ctypes.sizeof(kind))
        for field, _ in kind._fields_:
            lines.append(f'  printf("%zu\\n", offsetof({name}, {field}));')
            want.append(getattr(kind, field).offset)
    source, binary = tmp_path / "sizes.c", tmp_path / "sizes"
    source.write_text("\n".join(lines + ["  return 0;", "}"]))
    subprocess.run(["gcc", "-std=c11", str(source), "-o", str(binary)], check=True)
    assert [int(x) for x in subprocess.run([str(binary)], check=True, capture_output=True, text=True).stdout.split()] == want


# ------------------------------------------------------------------------------------------------ bookkeeping
def cache(**changes):
    return DensePagedCache(**{**dict(layers=2, kv_heads=2, head_dim=64, pages=6, max_requests=2, max_tokens=70, page_tokens=16, device="cpu"), **changes})


def test_pages_and_slots_are_handed_out_and_given_back():
    c = cache()
    assert c.admit("a") != c.admit("b") and c.free_pages == 6 and c.lengths.tolist() == [0, 0]
    with pytest.raises(RuntimeError, match="no free slot"):
        c.admit("c")
    with pytest.raises(ValueError, match="already"):
        c.admit("a")
    step = c.begin_prompt(["b", "a"], [17, 33])
    assert c.free_pages == 1 and step.cu_seqlens.tolist() == [0, 17, 50] and c.lengths.tolist() == [0, 0]
    step.finish()
    with pytest.raises(RuntimeError, match="finished"):
        step.finish()
    assert (c.tokens("a"), c.tokens("b")) == (33, 17)
    a = c.slot("a")
    assert c.lengths[a] == 33 and c.seen[a] == 33 and c.positions[1, a, 1, :33].tolist() == list(range(33))
    assert sorted(c.block_table[a, :3].tolist() + c.block_table[c.slot("b"), :2].tolist()) == sorted(c._pages[0] + c._pages[1])
    more = c.begin_prompt(["b"], [16])         # behind what it holds
    assert c.free_pages == 0 and more.cu_seqlens.tolist() == [0, 16] and more.cu_seqlens_k.tolist() == [0, 33]
    more.finish()
    for _ in range(15):
        c.begin_decode()
        c.advance()
    assert c.tokens("a") == 48 and c.positions[0, a, 0, 47] == 47
    with pytest.raises(RuntimeError, match="no free pages"):
        c.begin_decode()
    c.release("b")
    assert c.free_pages == 3 and c.lengths[a] == 48 and (c.lengths < 0).sum() == 1
    with pytest.raises(KeyError):
        c.tokens("b")
    assert c.admit("d") != a and c.tokens("d") == 0


def test_the_cache_refuses():
    for changes in (dict(layers=0), dict(pages=0), dict(page_tokens=0), dict(max_tokens=0)):
        with pytest.raises(ValueError):
            cache(**changes)
    for changes in (dict(head_dim=96), dict(dtype=torch.float32)):
        with pytest.raises(NotImplementedError):
            cache(**changes)
    c = cache()
    c.admit("a")
    for requests, tokens in ((["a", "a"], [1, 1]), (["a"], [0]), (["a"], [1, 2]), ([], []), (["a"], [71])):
        with pytest.raises(ValueError):
            c.begin_prompt(requests, tokens)
    with pytest.raises(KeyError):
        c.begin_prompt(["b"], [1])
    step = c.begin_prompt(["a"], [3])
    with pytest.raises(ValueError):
        step.attend(0, torch.zeros(3, 4, 64, dtype=BF16), torch.zeros(2, 2, 64, dtype=BF16), torch.zeros(2, 2, 64, dtype=BF16))
    c.release("a")
    with pytest.raises(RuntimeError, match="changed"):
        step.finish()
    c.admit("a")
    step = c.begin_prompt(["a"], [16])
    other = c.begin_prompt(["a"], [2])
    step.finish()
    with pytest.raises(RuntimeError, match="changed"):
        other.finish()
    assert c.block_table[c.slot("a"), 1:].tolist() == [-1] * 4
    with pytest.raises(RuntimeError, match="begin_decode"):
        c.advance()
    with pytest.raises(ValueError):
        c.evict(4, sink=4, recent=1)
    with pytest.raises(RuntimeError, match="without weights"):
        cache(weights=False).evict(4, sink=0, recent=0)
    c.evict(64, sink=4, recent=32)              # nothing to evict: nothing is launched
    assert c.free_pages == 5




def test_pages_that_cannot_all_be_had_are_not_reserved_at_all():
    c = cache(pages=3)
    a, b = c.admit("a"), c.admit("b")
    with pytest.raises(RuntimeError, match="no free pages"):
        c.begin_prompt(["a", "b"], [16, 48])
    with pytest.raises(ValueError, match="max_tokens"):
        c.begin_prompt(["a", "b"], [16, 71])
    assert c.free_pages == 3 and (c.block_table == -1).all()
    c.begin_prompt(["a", "b"], [16, 32]).finish()
    with pytest.raises(RuntimeError, match="no free pages"):
        c.begin_decode()
    c.release("b")
    assert (c.block_table[b] == -1).all() and c.block_table[a, 0] >= 0
    c.begin_decode()
    assert c.block_table[a, :2].tolist() == c._pages[a] and c.free_pages == 1


def test_a_step_does_not_outlive_its_pages(monkeypatch):
    c = cache()
    c.admit("a")
    step = c.begin_prompt(["a"], [16])
    c.release("a")
    assert c.admit("a") == step.slots[0]        # the same slot, as empty as it was, and without the step's page
    rows = torch.zeros(16, 2, 64, dtype=BF16)
    for call in (step.finish, lambda: step.attend(0, rows, rows, rows)):
        with pytest.raises(RuntimeError, match="changed"):
            call()
    c.admit("b")
    c.begin_prompt(["b"], [40]).finish()
    step = c.begin_prompt(["a"], [16])
    monkeypatch.setattr("inquant.dense_paged.evict_tokens", lambda *_, out_lengths, **__: out_lengths.copy_(c.lengths.clamp(max=32)))
    c.evict(32, sink=0, recent=0)               # gives back what lies behind every request's tokens
    with pytest.raises(RuntimeError, match="changed"):
        step.finish()


def test_rows_of_another_length_are_refused_before_they_are_stored():
    c = cache()
    c.admit("a")
    step = c.begin_prompt(["a"], [3])
    c.key_pages.fill_(7)
    rows = torch.zeros(3, 2, 64, dtype=BF16)
    with pytest.raises(ValueError, match="query"):
        step.attend(0, torch.zeros(2, 4, 64, dtype=BF16), rows, rows)
    assert (c.key_pages == 7).all()


def cut(c, budget, monkeypatch):
    monkeypatch.setattr("inquant.dense_paged.evict_tokens", lambda *_, out_lengths, **__: out_lengths.copy_(c.lengths.clamp(max=budget)))
    c.evict(budget, sink=0, recent=0)


def refused_and_repeated(c):
    """``advance`` refuses and changes nothing; the step begun again is taken into account."""
    held, seen, lengths, positions = list(c._held), list(c._seen), c.lengths.clone(), c.positions.clone()
    with pytest.raises(RuntimeError, match="begin_decode"):
        c.advance()
    assert (c._held, c._seen) == (held, seen) and torch.equal(c.lengths, lengths) and torch.equal(c.positions, positions)
    c.begin_decode()
    c.advance()
    assert all(c._held[s] == held[s] + 1 for s in c._slots.values())


def test_a_step_whose_token_was_evicted_is_not_counted(monkeypatch):
    c = cache()
    c.admit("a")
    c.begin_prompt(["a"], [40]).finish()
    c.begin_decode()
    cut(c, 35, monkeypatch)                      # does not end a page: there is room behind it, for a token that is not there
    refused_and_repeated(c)


def test_a_step_whose_place_was_given_back_is_not_counted(monkeypatch):
    c = cache()
    c.admit("a"), c.admit("b")
    c.begin_prompt(["a", "b"], [16, 40]).finish()
    c.begin_decode()
    cut(c, 33, monkeypatch)                      # of "a" nothing leaves but the page of its next token
    refused_and_repeated(c)


def test_a_request_that_came_in_during_a_step_is_not_counted():
    c = cache()
    c.admit("a")
    c.begin_prompt(["a"], [5]).finish()
    c.begin_decode()
    c.admit("b")
    c.begin_prompt(["b"], [7]).finish()
    refused_and_repeated(c)
    assert (c.tokens("a"), c.tokens("b")) == (6, 8)


def test_a_chunk_that_came_in_during_a_step_ends_it():
    c = cache()
    c.admit("a")
    c.begin_prompt(["a"], [5]).finish()
    c.begin_decode()
    c.begin_prompt(["a"], [4]).finish()
    refused_and_repeated(c)


def test_a_slot_that_changed_hands_during_a_step_is_not_counted():
    c = cache()
    c.admit("a"), c.admit("b")
    c.begin_prompt(["a", "b"], [5, 5]).finish()
    c.begin_decode()
    c.release("b")
    assert c.admit("b") >= 0
    c.begin_prompt(["b"], [5]).finish()          # as many tokens as before, others
    refused_and_repeated(c)


def test_a_step_is_counted_once():
    c = cache()
    c.admit("a")
    c.begin_prompt(["a"], [5]).finish()
    c.begin_decode()
    c.advance()
    refused_and_repeated(c)


def test_what_does_not_touch_a_step_does_not_end_it(monkeypatch):
    c = cache(pages=9, max_requests=3)
    for r in "abc":
        c.admit(r)
    c.begin_prompt(["a", "b", "c"], [5, 16, 20]).finish()
    c.begin_decode()
    c.evict(64, sink=4, recent=32)               # nobody holds so many
    c.begin_prompt(["a"], [30])                  # pages are reserved behind the step's, nothing else has happened
    c.release("c")                               # a request that has ended
    with pytest.raises(KeyError):
        c.begin_prompt(["z"], [1])
    c.advance()
    assert (c.tokens("a"), c.tokens("b")) == (6, 17)
    # without begin_decode, where the last page has room: the step begins with its first layer
    monkeypatch.setattr("inquant.dense_paged.paged_attention", lambda q, *_, **__: (q, None))
    q, k = torch.zeros(3, 4, 64, dtype=BF16), torch.zeros(3, 2, 64, dtype=BF16)
    for layer in range(2):
        c.decode(layer, q, k, k)
    c.advance()
    assert (c.tokens("a"), c.tokens("b")) == (7, 18)
    c.decode(0, q, k, k)
    c.admit("d")
    with pytest.raises(RuntimeError, match="begin_decode"):
        c.advance()


@pytest.mark.parametrize("call,name,shape,dtype", [
    (prompt_attention, "out", (8, 4, 128), BF16), (prompt_attention, "lse", (4, 8), torch.float32), (prompt_weights, "out", (2, 8), torch.float32),
    (paged_attention, "out", (3, 4, 128), BF16), (paged_attention, "weights", (3, 2, 32), torch.float32),
    (paged_attention, "out_weights", (3, 2, 32), torch.float32), (evict_tokens, "out_weights", (3, 2, 32), torch.float32),
    (evict_tokens, "out_positions", (3, 2, 32), torch.int32)])
def test_results_whose_rows_share_memory_are_refused(no_device, monkeypatch, call, name, shape, dtype):
    monkeypatch.setattr(torch.cuda, "device", lambda _device: contextlib.nullcontext())
    case = dict(paged_case() if call is paged_attention else evict_case() if call is evict_tokens else prompt_case())
    if call is prompt_weights:
        case["lse"] = torch.zeros(4, 8)
        del case["value"]
    for axis in range(len(shape) - 1):
        row = torch.zeros([1 if i == axis else n for i, n in enumerate(shape)], dtype=dtype)
        views = [row.expand(shape)]                                            # the same row for all
        if axis == 0:
            step = [shape[-1] // 2] + [shape[-1]] * (len(shape) - 2) + [1]         # rows that begin inside the one before
            views.append(torch.zeros(4096, dtype=dtype).as_strided(shape, step))
        for view in views:
            with pytest.raises(ValueError, match=name):
                call(**{**case, name: view})
    room = torch.zeros([2 * n for n in shape], dtype=dtype)[tuple(slice(n, None) for n in shape)]
    for view in (room, torch.zeros(shape[::-1][1:] + shape[-1:], dtype=dtype).transpose(0, 1) if len(shape) == 3 else room):
        with pytest.raises(pytest.fail.Exception, match="not refused"):        # gaps and other orders of rows are served
            call(**{**case, name: view})
    if name == "weights":                                                      # read alone, they may be the same row for all
        with pytest.raises(pytest.fail.Exception, match="not refused"):
            call(**{**case, name: torch.zeros(1, 1, 32).expand(shape), "out_weights": torch.zeros(shape)})


@pytest.mark.parametrize("changes", [dict(query=torch.zeros(3, 4, 64)), dict(query=torch.zeros(3, 4, 64, dtype=torch.float16)),
                                     dict(query=torch.zeros(3, 4, 128, dtype=BF16)), dict(query=torch.zeros(3, 5, 64, dtype=BF16)),
                                     dict(query=torch.zeros(3, 0, 64, dtype=BF16)), dict(scale=0.0), dict(scale=float("nan")), dict(window=0), dict(window=-1),
                                     dict(query=torch.zeros(3, 4, 64, dtype=BF16, device="meta")), dict(key=torch.zeros(3, 2, 64, dtype=BF16, device="meta")),
                                     dict(value=torch.zeros(3, 2, 64, dtype=BF16, device="meta"))])
@pytest.mark.parametrize("weights", [True, False])
def test_what_a_prompt_step_refuses_is_not_stored(no_device, weights, changes):
    if "window" in changes and not weights:
        changes = dict(scale=-1.0)                # there are no weights that a window would be of
    c = cache(weights=weights)
    c.admit("a")
    step = c.begin_prompt(["a"], [3])
    c.key_pages.fill_(7), c.value_pages.fill_(7)
    rows = torch.zeros(3, 2, 64, dtype=BF16)
    with pytest.raises((ValueError, NotImplementedError)):
        step.attend(0, **{**dict(query=torch.zeros(3, 4, 64, dtype=BF16), key=rows, value=rows), **changes})
    assert (c.key_pages == 7).all() and (c.value_pages == 7).all()
