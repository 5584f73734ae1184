"""What the operators over the cache hand to their launchers, looked at without a GPU: scratch, its parts and their addresses."""
import itertools

import pytest
import torch

from railgun_b200 import ops


class Called(Exception):
    pass


@pytest.fixture
def calls(monkeypatch):
    """Runs an operator on CPU tensors up to its launch: its arguments as numbers, and the scratch as (address, bytes)."""
    made, empty = [], torch.empty

    def scratch(*a, **k):
        t = empty(*a, **k)
        made.append(t)
        return t

    def launcher(lib, name):
        def call(*args):
            raise Called(args)
        return call

    def address(t):
        return 0 if t is None else t.data_ptr()
    for name in ("_check_rows", "_check_out_view", "_check"):
        monkeypatch.setattr(ops, name, lambda *a, **k: None)
    for name in ("c_int", "c_float", "c_void_p"):
        monkeypatch.setattr(ops, name, lambda v: 0 if v is None else v)
    monkeypatch.setattr(ops, "_ptr", address)
    monkeypatch.setattr(ops, "_fn", launcher)
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    monkeypatch.setattr(ops, "num_sms", lambda device: 148)
    monkeypatch.setattr(ops, "_tc_error_flag", lambda device: None)
    monkeypatch.setattr(torch, "empty", scratch)

    def run(f, *a, **k):
        made.clear()
        with pytest.raises(Called) as e:
            f(*a, **k)
        return e.value.args[0], [(t.data_ptr(), t.numel() * t.element_size()) for t in made]
    return run


def tensors(T, nh, nkv, d, page, dtype, lists, pages):
    q = torch.zeros(T, nh * d, dtype=dtype)
    kv = torch.zeros(4, 2, nkv, page, d, dtype=dtype)
    table = torch.zeros(lists, pages, dtype=torch.int32)
    return q, torch.zeros_like(q), kv, table


# rows, query heads, kv heads, head size
SIZES = [(199, 3, 1, 33), (201, 3, 3, 5), (601, 1, 1, 5), (593, 1, 1, 255), (197, 5, 5, 7), (199, 3, 1, 128), (601, 1, 1, 64), (2, 40, 1, 1),
         (211, 9, 3, 130)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,nh,nkv,d", SIZES)
def test_parts_lie_where_their_loads_can_read_them(calls, T, nh, nkv, d, dtype):
    """(m, l) of a part are read two at a time, its outputs and the scores four at a time where they come in fours."""
    page, seen = 16, 0
    for longest, own in itertools.product((0, 500, 600, 3001), (0, 100, 450, 2000)):
        q, out, kv, table = tensors(T, nh, nkv, d, page, dtype, T, 256)
        pos, slots = torch.zeros(T, dtype=torch.int32), torch.arange(T, dtype=torch.int32)
        args, made = calls(ops.prefix_attention, q, out, kv, table[:1], torch.tensor([[0, T, longest]], dtype=torch.int32), table, pos, nh, nkv, d,
                           0.125, max_rows=T, max_prefix=longest, max_own=own)
        if made:
            (at, size), = made
            part_o, part_ml = next((args[i], args[i + 1]) for i in range(len(args)) if args[i] == at)
            seen += 1
            parts = (size // 4 - (part_ml - at) // 4) // 2
            assert part_o % 16 == 0 and part_ml % 8 == 0 and parts % (T * nh) == 0 and part_o + 4 * parts * d <= part_ml
        if own == 0:
            continue
        weights = torch.zeros(1, nkv, own)
        args, made = calls(ops.weighed_attention, q, out, kv, weights, slots, table, pos, nh, nkv, d, 0.125, max_context=own)
        if made:
            (at, size), = made
            i = next(i for i in range(len(args)) if args[i] == at)
            scores, (part_o, part_ml) = args[i], args[i - 2:i]
            if part_o:
                seen += 1
                parts = (at + size - part_ml) // 8
                assert scores % 16 == 0 and part_o % 16 == 0 and part_ml % 8 == 0
                assert parts % (T * nh) == 0 and part_o + 4 * parts * d <= part_ml and scores + 4 * T * nh * own <= part_o
    assert seen or T == 2


@pytest.mark.parametrize("n", [-1, 1 << 31, 1 << 32, (1 << 32) + 5, 1 << 63])
@pytest.mark.parametrize("operator,name", [(o, n) for o, names in dict(
    prefix="max_rows max_prefix max_own", weigh="max_context", prompt="max_rows max_context", evict="max_context protect_first protect_last").items()
    for n in names.split()])
def test_counts_that_no_launcher_can_take(calls, operator, name, n):
    """A launcher's counts are 32-bit: a larger one would arrive as another number, and the call do nothing, or something else."""
    q, out, kv, table = tensors(3, 2, 1, 16, 8, torch.float32, 3, 4)
    weights, places = torch.zeros(3, 1, 32), torch.zeros(3, 1, 32, dtype=torch.int32)
    ints = torch.zeros(3, dtype=torch.int32)
    if operator == "prefix":
        f, args, counts = ops.prefix_attention, (q, out, kv, table[:0], torch.zeros(0, 3, dtype=torch.int32), table, ints, 2, 1, 16, 0.25), dict(
            max_rows=0, max_prefix=0, max_own=32)
    elif operator == "weigh":
        f, args, counts = ops.weighed_attention, (q, out, kv, weights, ints, table, ints, 2, 1, 16, 0.25), dict(max_context=32)
    elif operator == "prompt":
        f, args, counts = ops.prompt_key_weights, (q, kv, weights, ints, table, torch.zeros(4, dtype=torch.int32), ints, ints, 2, 1, 16, 0.25), dict(
            max_rows=1, max_context=32)
    else:
        f, args, counts = ops.evict_entries, (kv, weights, places, weights, places, ints, table, ints, ints, ints, 1, 16), dict(
            protect_first=1, protect_last=1, max_context=32)
    calls(f, *args, **counts)                                          # as it is, it gets to its launcher
    with pytest.raises(ops.KernelError):
        f(*args, **{**counts, name: n})
