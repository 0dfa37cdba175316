"""The operators of a step whose sequences take any number of tokens, through the C ABI (step plans, stored rows, attention of
chunks over pages, sampling), against plain 64-bit implementations, and their refusals. Refusals are decided on the host, so
they run without a GPU."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

from chroma_amd._src import native

gpu = pytest.mark.gpu
BOTH = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
DTYPES = {torch.float32: native.FLOAT32, torch.bfloat16: native.BFLOAT16}
HALF = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8}  # half a step relative to a value


def pointer(tensor):
    return None if tensor is None else tensor.data_ptr()


def queue(name, call, stream=None):
    error = ctypes.create_string_buffer(256)
    native.check(getattr(native.library(), name)(ctypes.byref(call), stream, error, len(error)), error)


def queue_in(name, call, stream=None, workspace=None):
    """A call that takes a workspace; returns it."""
    lib, error = native.library(), ctypes.create_string_buffer(256)
    if workspace is None:
        workspace = torch.full((max(1, getattr(lib, name + "_workspace")(ctypes.byref(call))),), 0xAB, dtype=torch.uint8, device="cuda")
    native.check(getattr(lib, name)(ctypes.byref(call), workspace.data_ptr(), workspace.numel(), stream, error, len(error)), error)
    return workspace


def on_gpu(inputs):
    return {name: value.cuda() if isinstance(value, torch.Tensor) else value for name, value in inputs.items()}


# ------------------------------------------------------------------------------------------------ step plans
def plan_reference(lengths, counts, table, free, cursor, *, tokens, pages, page):
    """Sequence by sequence, token by token."""
    span = table.shape[1]
    table, room = [list(row) for row in table.tolist()], span * page
    cursor = max(0, cursor)
    starts, slots, positions, owners, after = [0], [], [], [], []
    for b, (length, count) in enumerate(zip(lengths, counts)):
        length, count = min(max(0, length), room), min(max(0, count), tokens - len(slots))
        for p in range(length, length + count):
            if p < room and p % page == 0:
                table[b][p // page] = int(free[cursor]) if cursor < len(free) else -1
                cursor += 1
            at = table[b][p // page] if p < room else -1
            slots.append(at * page + p % page if 0 <= at < pages else -1)
            positions.append(p)
            owners.append(b)
        starts.append(len(slots))
        after.append(min(length + count, room))
    behind = [-1] * (tokens - len(slots))
    return {"table": table, "starts": starts, "slots": slots + behind, "positions": positions + behind, "owners": owners + behind,
            "new_lengths": after, "taken": [cursor]}


def plan_call(inputs, made, *, tokens, pages, page, optional=True):
    n, span = inputs["table"].shape
    return native.PagedPlan(
        lengths=pointer(inputs["lengths"]), counts=pointer(inputs["counts"]), free_pages=pointer(inputs["free"]) if len(inputs["free"]) else None,
        cursor=pointer(inputs["cursor"]), table=pointer(inputs["table"]), starts=pointer(made["starts"]), slots=pointer(made["slots"]),
        positions=pointer(made["positions"]) if optional else None, owners=pointer(made["owners"]) if optional else None,
        new_lengths=pointer(made["new_lengths"]) if optional else None, taken=pointer(made["taken"]), sequences=n, tokens=tokens, pages=pages,
        page_rows=page, span=span, table_stride=inputs["table"].stride(0), free_count=len(inputs["free"]))


def plan_room(n, tokens):
    return {name: torch.full((size,), -77, dtype=torch.int64, device="cuda") for name, size in
            (("starts", n + 1), ("slots", tokens), ("positions", tokens), ("owners", tokens), ("new_lengths", n), ("taken", 1))}


def plan_inputs(lengths, counts, *, page, span, pages, free, cursor=0, seed=0):
    g = torch.Generator().manual_seed(seed)
    table = torch.full((len(lengths), span), -1, dtype=torch.int64)
    order, taken = torch.randperm(pages, generator=g), 0
    for b, n in enumerate(lengths):
        for i in range(min(span, -(-max(0, n) // page))):
            table[b, i] = order[taken]
            taken += 1
    return {"lengths": torch.tensor(lengths), "counts": torch.tensor(counts), "table": table, "free": order[taken: taken + free],
            "cursor": None if cursor is None else torch.tensor([cursor])}


def check_plan(inputs, *, tokens, pages, page, optional=True):
    want = plan_reference(inputs["lengths"].tolist(), inputs["counts"].tolist(), inputs["table"], inputs["free"],
                          0 if inputs["cursor"] is None else int(inputs["cursor"]), tokens=tokens, pages=pages, page=page)
    device, made = on_gpu(inputs), plan_room(len(inputs["lengths"]), tokens)
    queue("chroma_hip_paged_plan", plan_call(device, made, tokens=tokens, pages=pages, page=page, optional=optional))
    got = {**{name: value.tolist() for name, value in made.items()}, "table": device["table"].tolist()}
    for name in want:
        if optional or name not in ("positions", "owners", "new_lengths"):
            assert got[name] == want[name], name
        else:
            assert set(got[name]) == {-77}, name
    return want


PLANS = [  # (lengths, counts, page, span, free, cursor, tokens)
    ([0], [1], 16, 1, 1, 0, 1),
    ([5], [1], 16, 1, 0, None, 1),
    ([16, 15, 0, 17, 31], [1, 1, 1, 1, 1], 16, 4, 9, 2, 5),
    ([0, 0, 0], [0, 0, 0], 16, 2, 3, 0, 4),
    ([3, 100, 0, 7], [40, 0, 33, 1], 12, 12, 40, 5, 100),
    ([0, 9, 0, 0, 5], [0, 0, 700, 0, 1], 1, 720, 800, 3, 800),
    ([7, 1, 2], [3, 9, 4], 7, 3, 2, 0, 16),  # too few free pages
    ([7, 1, 2], [30, 9, 4], 7, 3, 30, 0, 50),  # more rows than the table row has pages for
    ([40, 2, 2], [30, 9, 4], 7, 3, 30, 0, 20),  # lengths behind it; the step has room for fewer tokens
    ([-5, 2, 2**40], [-3, 5, 2], 7, 3, 30, -4, 20),
    ([1, 2, 3], [2**62, 2**62, 2**62], 16, 40, 100, 0, 333),
]


@gpu
@pytest.mark.parametrize("plan", PLANS, ids=range(len(PLANS)))
def test_plan(plan):
    lengths, counts, page, span, free, cursor, tokens = plan
    pages = 4 + free + sum(min(span, -(-max(0, n) // page)) for n in lengths)
    inputs = plan_inputs(lengths, counts, page=page, span=span, pages=pages, free=free, cursor=cursor)
    check_plan(inputs, tokens=tokens, pages=pages, page=page)
    check_plan(inputs, tokens=tokens, pages=pages, page=page, optional=False)


@gpu
@pytest.mark.parametrize("sequences,most", [(1023, 3), (1024, 40), (1025, 1), (2500, 7), (65535, 2)])
def test_plan_of_many_sequences(sequences, most):
    rng = np.random.default_rng(sequences)
    lengths, counts = rng.integers(0, 60, sequences).tolist(), rng.integers(0, most + 1, sequences).tolist()
    pages = sequences * 13
    inputs = plan_inputs(lengths, counts, page=8, span=13, pages=pages, free=sequences * 5, cursor=11)
    want = check_plan(inputs, tokens=sum(counts) + 300, pages=pages, page=8)
    assert want["taken"][0] > 11


@gpu
def test_plan_of_bad_pages_and_padded_rows():
    """A last page outside the cache gives no slot; what lies between the table's rows stays."""
    inputs = plan_inputs([20, 20, 20, 3], [5, 5, 20, 1], page=16, span=4, pages=50, free=9)
    inputs["table"][0, 1], inputs["table"][1, 1], inputs["free"][0] = 50, -9, 2**61
    room = torch.full((4, 9), 123, dtype=torch.int64)
    room[:, :4] = inputs["table"]
    inputs["table"] = room[:, :4]
    want = plan_reference([20, 20, 20, 3], [5, 5, 20, 1], inputs["table"], inputs["free"], 0, tokens=40, pages=50, page=16)
    assert want["slots"][:10] == [-1] * 10 and want["slots"][22:30] == [-1] * 8
    device, made = on_gpu({**inputs, "table": None}), plan_room(4, 40)
    room = room.cuda()
    device["table"] = room[:, :4]
    queue("chroma_hip_paged_plan", plan_call(device, made, tokens=40, pages=50, page=16))
    assert {name: value.tolist() for name, value in made.items()} == {name: value for name, value in want.items() if name != "table"}
    assert room[:, :4].tolist() == want["table"] and (room[:, 4:] == 123).all()


@gpu
def test_plans_follow_one_another_on_the_device():
    """Each step's lengths and cursor are the last one's, the free pages one list; replayed from two graphs that take turns."""
    page, span, pages, n, steps = 4, 30, 400, 9, 8
    counts = torch.tensor([1, 0, 3, 9, 1, 1, 2, 0, 4])
    free = torch.randperm(pages, generator=torch.Generator().manual_seed(5))
    state = on_gpu({"counts": counts, "free": free, "table": torch.full((n, span), -1), "cursor": torch.zeros(1, dtype=torch.int64),
                    "lengths": torch.zeros(n, dtype=torch.int64)})
    rooms = [plan_room(n, 24), plan_room(n, 24)]
    rooms[1]["new_lengths"].zero_()
    rooms[1]["taken"].zero_()
    graphs = []
    for one, other in ((0, 1), (1, 0)):
        inputs = {**state, "lengths": rooms[other]["new_lengths"], "cursor": rooms[other]["taken"]}
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            queue("chroma_hip_paged_plan", plan_call(inputs, rooms[one], tokens=24, pages=pages, page=page), torch.cuda.current_stream().cuda_stream)
        graphs.append(graph)
    lengths, cursor, table = [0] * n, 0, torch.full((n, span), -1)
    for step in range(steps):
        want = plan_reference(lengths, counts.tolist(), table, free, cursor, tokens=24, pages=pages, page=page)
        graphs[step % 2].replay()
        torch.cuda.synchronize()
        got = {name: value.tolist() for name, value in rooms[step % 2].items()}
        assert {**got, "table": state["table"].tolist()} == want
        lengths, cursor, table = want["new_lengths"], want["taken"][0], torch.tensor(want["table"])


def plain_plan_call(**changes):
    """A valid call on addresses that are never followed."""
    fields = dict(lengths=4096, counts=8192, free_pages=12288, cursor=16384, table=20480, starts=24576, slots=28672, positions=32768, owners=36864,
                  new_lengths=40960, taken=45056, sequences=4, tokens=16, pages=100, page_rows=16, span=8, table_stride=8, free_count=20)
    fields.update(changes)
    return native.PagedPlan(**fields)


@pytest.mark.parametrize("changes,message", [
    (dict(sequences=0), "sequences"), (dict(sequences=65536), "sequences"), (dict(tokens=0), "tokens"), (dict(tokens=2**24 + 1), "tokens"),
    (dict(pages=0), "pages"), (dict(pages=2**31), "pages"), (dict(page_rows=0), "page_rows"), (dict(span=0), "span"),
    (dict(span=2**20, table_stride=2**20, page_rows=2**11), "span"), (dict(table_stride=7), "table row"), (dict(free_count=-1), "extent"),
    (dict(free_count=2**50), "extent"), (dict(lengths=None), "null"), (dict(counts=None), "null"), (dict(free_pages=None), "null"),
    (dict(table=None), "null"), (dict(starts=None), "null"), (dict(slots=None), "null"), (dict(taken=None), "null"),
    (dict(new_lengths=4096), "overlaps"), (dict(taken=16384), "overlaps"), (dict(taken=16384 - 4), "overlaps"), (dict(slots=20480 + 8 * 31), "overlaps"),
    (dict(positions=28672 + 8 * 15), "overlaps"), (dict(starts=12288 + 8 * 19), "overlaps"), (dict(owners=32768), "overlaps"),
])
def test_plan_refusals(changes, message):
    with pytest.raises(RuntimeError, match="paged_plan.*" + message):
        queue("chroma_hip_paged_plan", plain_plan_call(**changes))


# ------------------------------------------------------------------------------------------------ stored rows
def store_call(keys, values, new_keys, new_values, slots, count=None):
    """keys and values [layers, rows, bytes], new ones [layers, count, bytes]."""
    layers, rows, row_bytes = keys.shape
    return native.CacheStore(keys=pointer(keys), values=pointer(values), new_keys=pointer(new_keys), new_values=pointer(new_values),
                             slots=pointer(slots), layers=layers, rows=rows, count=new_keys.shape[1] if count is None else count, row_bytes=row_bytes,
                             layer_pitch=keys.stride(0), new_layer_pitch=new_keys.stride(0), new_row_pitch=new_keys.stride(1))


def noise(*shape, seed=0):
    return torch.randint(0, 256, shape, dtype=torch.uint8, generator=torch.Generator().manual_seed(seed))


@gpu
@pytest.mark.parametrize("layers,rows,count,row_bytes", [(1, 1, 1, 1), (3, 10, 4, 15), (2, 300, 300, 16), (24, 700, 65, 1024), (1, 50, 7, 1000),
                                                         (2, 9, 5, 100003), (1, 3000, 2999, 33), (5, 40, 11, 4096)])
@pytest.mark.parametrize("offset,extra", [(0, 0), (16, 48), (1, 3)], ids=["plain", "columns", "unaligned"])
def test_store(layers, rows, count, row_bytes, offset, extra):
    """Columns of a wider matrix, rows without a slot, rows that no slot names."""
    g = torch.Generator().manual_seed(rows)
    slots = torch.randperm(rows, generator=g)[:count].clone()
    slots[torch.rand(count, generator=g) < 0.2] = torch.tensor([-1, -(2**62), rows, 2**62])[torch.randint(0, 4, (), generator=g)]
    wide = noise(layers, count, 2 * row_bytes + extra, seed=1)
    cache = noise(2, layers * rows * row_bytes + offset, seed=2)
    want = cache.clone()
    for which in range(2):
        view = want[which, offset:].view(layers, rows, row_bytes)
        for i, slot in enumerate(slots.tolist()):
            if 0 <= slot < rows:
                view[:, slot] = wide[:, i, which * row_bytes: (which + 1) * row_bytes]
    wide, device = wide.cuda(), cache.cuda()
    keys, values = (device[which, offset:].view(layers, rows, row_bytes) for which in range(2))
    queue("chroma_hip_cache_store", store_call(keys, values, wide[:, :, :row_bytes], wide[:, :, row_bytes: 2 * row_bytes], slots.cuda()))
    assert torch.equal(device.cpu(), want)


@gpu
def test_store_of_nothing_and_past_32_bits():
    keys, values = (torch.zeros(1, (1 << 22) + 5, 1040, dtype=torch.uint8, device="cuda") for _ in range(2))  # 4.4 GB each
    new = noise(2, 3, 1040).cuda()
    slots = torch.tensor([1 << 22, 7, (1 << 22) + 4], device="cuda")
    queue("chroma_hip_cache_store", store_call(keys, values, new[:1], new[1:], slots, count=0))
    assert not keys.view(-1, 1040)[slots].any()
    queue("chroma_hip_cache_store", store_call(keys, values, new[:1], new[1:], slots))
    assert torch.equal(keys[0, slots], new[0]) and torch.equal(values[0, slots], new[1])
    assert int(keys[0].any(1).sum()) == 3


def plain_store_call(**changes):
    fields = dict(keys=1 << 20, values=2 << 20, new_keys=3 << 20, new_values=(3 << 20) + 64, slots=4 << 20, layers=2, rows=100, count=10, row_bytes=64,
                  layer_pitch=6400, new_layer_pitch=1280, new_row_pitch=128)
    fields.update(changes)
    return native.CacheStore(**fields)


@pytest.mark.parametrize("changes,message", [
    (dict(layers=0), "layers"), (dict(layers=32768), "layers"), (dict(row_bytes=0), "rows of"), (dict(rows=0), "rows"), (dict(rows=2**32), "rows"),
    (dict(count=-1), "count"), (dict(count=2**32), "count"), (dict(layer_pitch=-1), "pitch"), (dict(new_row_pitch=2**47), "pitch"),
    (dict(layer_pitch=6399), "smaller"), (dict(new_row_pitch=63), "smaller"), (dict(keys=None), "null"), (dict(values=None), "null"),
    (dict(new_keys=None), "null"), (dict(new_values=None), "null"), (dict(slots=None), "null"), (dict(values=(1 << 20) + 12799), "overlap"),
    (dict(new_keys=(1 << 20) + 12799), "overlap"), (dict(new_values=(2 << 20) - 1200), "overlap"), (dict(slots=(2 << 20) + 64), "overlap"),
    (dict(keys=1 << 20, values=(1 << 20) + 6400, layer_pitch=12800), "overlap"),
])
def test_store_refusals(changes, message):
    with pytest.raises(RuntimeError, match="cache_store.*" + message):
        queue("chroma_hip_cache_store", plain_store_call(**changes))


# ------------------------------------------------------------------------------------------------ attention of chunks
def chunk_call(q, k_pages, v_pages, table, lengths, starts, out, *, k_new=None, v_new=None, sinks=None, longest=None, window=0, first=0,
               scale=None, heads_first=False):
    """The call for tensors: q and out [T, KV, G, D], pages [P, R, KV, D] (or [P, KV, R, D])."""
    tokens, kv, group, dim = q.shape
    rows = k_pages.shape[2 if heads_first else 1]
    row_stride, head_stride = k_pages.stride()[2 if heads_first else 1], k_pages.stride()[1 if heads_first else 2]
    return native.PagedChunk(
        q=pointer(q), k_pages=pointer(k_pages), v_pages=pointer(v_pages), k_new=pointer(k_new), v_new=pointer(v_new), sinks=pointer(sinks),
        table=pointer(table), lengths=pointer(lengths), starts=pointer(starts), out=pointer(out), tokens=tokens, sequences=len(lengths), kv_heads=kv,
        group=group, dim=dim, pages=k_pages.shape[0], page_rows=rows, page_stride=k_pages.stride()[0], row_stride=row_stride,
        head_stride=head_stride, q_stride=q.stride()[0], new_stride=0 if k_new is None else k_new.stride()[0], out_stride=out.stride()[0],
        table_stride=table.stride()[0], longest=table.shape[1] * rows if longest is None else longest, window=window, first=first,
        scale=dim**-0.5 if scale is None else scale, dtype=DTYPES[q.dtype])


def chunk_reference(q, k_pages, v_pages, table, lengths, starts, *, k_new=None, v_new=None, sinks=None, longest=None, window=0, first=0, scale=None):
    """(result in 64 bits, bound of a float evaluation rounded once to q's type, which tokens a sequence has), token by token.

    The bound: a score's products and sum, (D + 3) roundings of at most sum |q k|; a weight's exponential, 1.2e-7 + 6e-8 |x|
    relative; a sum of n weighted values in any order, n roundings of at most sum p |v|; for bfloat16 also the weight's
    rounding, half a step of it; and half a step of the result."""
    tokens, kv, group, dim = q.shape
    dtype, rows = q.dtype, k_pages.shape[1]
    longest = table.shape[1] * rows if longest is None else longest
    scale = dim**-0.5 if scale is None else scale
    result, bound = torch.zeros(tokens, kv, group, dim, dtype=torch.float64), torch.zeros(tokens, kv, group, dim, dtype=torch.float64)
    taken = torch.zeros(tokens, dtype=torch.bool)
    for b in range(len(lengths)):
        begin = min(max(int(starts[b]), 0), tokens)
        end = min(max(int(starts[b + 1]), begin), tokens)
        taken[begin:end] = True
        length = min(max(int(lengths[b]), 0), longest)
        where = [(j, int(table[b, j // rows])) for j in range(length)]
        where = [(j, page) for j, page in where if 0 <= page < k_pages.shape[0]]
        places = torch.tensor([page * rows + j % rows for j, page in where], dtype=torch.int64)
        cached_k, cached_v = (x.reshape(-1, kv, dim)[places].double() for x in (k_pages, v_pages))
        position = torch.tensor([j for j, _ in where], dtype=torch.int64)
        if k_new is not None:
            cached_k, cached_v = torch.cat([cached_k, k_new[begin:end].double()]), torch.cat([cached_v, v_new[begin:end].double()])
            position = torch.cat([position, length + torch.arange(end - begin)])
        for i in range(end - begin):
            now = length + i if k_new is not None else length - (end - begin) + i
            seen = position <= now
            if window:
                seen &= (position > now - window) | (position < first)
            if not seen.any():
                continue
            k, v = cached_k[seen], cached_v[seen]
            token = q[begin + i].double()  # [KV, G, D]
            products = token[:, :, None] * k.transpose(0, 1)[:, None]  # [KV, G, S, D]
            s = products.sum(-1) * scale
            off = (dim + 3) * 2.0**-24 * products.abs().sum(-1).amax(-1) * abs(scale)  # [KV, G]
            joined = s if sinks is None else torch.cat([s, sinks.double().view(kv, group, 1)], 2)
            p = torch.softmax(joined, 2)[:, :, : len(k)]
            result[begin + i] = p @ v.transpose(0, 1)
            reach = (joined.amax(2, keepdim=True) - joined)[torch.isfinite(joined)].amax().clamp(max=90.0)
            relative = 2 * off + 2 * (1.2e-7 + 6e-8 * float(reach)) + 2 * (len(k) + 8) * 2.0**-24
            spread = p @ v.transpose(0, 1).abs()
            bound[begin + i] = relative[:, :, None] * v.abs().amax(0)[:, None] + (HALF[dtype] * spread if dtype == torch.bfloat16 else 0.0)
    return result, bound + HALF[dtype] * result.abs() + 1e-37, taken


def chunk_inputs(counts, lengths, *, kv, group, dim, page, dtype, fresh=True, sinks=True, seed=0, spread=1.0, behind=2):
    """CPU tensors; pages in random order, rows behind a sequence's last and unused pages hold NaN and infinities, and so do
    the rows of q and of the new keys and values that no sequence has."""
    g = torch.Generator().manual_seed(seed)
    span = max(1, -(-max(lengths) // page))
    used = [-(-max(0, n) // page) for n in lengths]
    pages, tokens = sum(used) + 3, sum(counts) + behind
    order, taken = torch.randperm(pages, generator=g), 0
    table = torch.full((len(lengths), span), -1, dtype=torch.int64)

    def values(*shape):
        return (torch.randn(*shape, generator=g) * spread).to(dtype)

    k = torch.full((pages, page, kv, dim), math.nan, dtype=dtype)
    v = torch.full((pages, page, kv, dim), math.inf, dtype=dtype)
    for b, n in enumerate(lengths):
        for i in range(used[b]):
            table[b, i] = order[taken]
            rows = min(page, n - i * page)
            k[order[taken], :rows], v[order[taken], :rows] = values(rows, kv, dim), values(rows, kv, dim)
            taken += 1
    inputs = {"q": values(tokens, kv, group, dim), "k_pages": k, "v_pages": v, "table": table, "lengths": torch.tensor(lengths, dtype=torch.int64),
              "starts": torch.tensor([0] + np.cumsum(counts).tolist(), dtype=torch.int64), "k_new": values(tokens, kv, dim) if fresh else None,
              "v_new": values(tokens, kv, dim) if fresh else None, "sinks": values(kv * group) if sinks else None}
    for name in ("q", "k_new", "v_new"):
        if inputs[name] is not None:
            inputs[name][sum(counts):] = math.nan
    return inputs


def check_chunk(inputs, **options):
    want, bound, taken = chunk_reference(**inputs, **options)
    device = on_gpu(inputs)
    out = torch.full(device["q"].shape, 7.0, dtype=device["q"].dtype, device="cuda")
    queue_in("chroma_hip_paged_chunk_attention", chunk_call(**device, out=out, **options))
    got = out.cpu().double()
    assert (got[~taken] == 7.0).all()
    fine = torch.isfinite(want)
    assert torch.equal(got.isnan()[taken], want.isnan()[taken]) and torch.equal(got[taken][~fine[taken]].nan_to_num(0.5), want[taken][~fine[taken]].nan_to_num(0.5))
    excess = torch.where(fine, (got - want).abs() - bound, 0.0)[taken].amax()
    assert excess <= 0, f"off by {float(torch.where(fine, got - want, 0.0)[taken].abs().amax())}, {float(excess)} more than the bound"
    return out


CHUNKS = [  # (tokens, cached rows, kv, group, dim, page)
    ([1], [0], 1, 1, 8, 1),
    ([1, 0, 3, 17], [0, 5, 2, 64], 2, 3, 16, 16),
    ([16], [113], 2, 8, 64, 16),
    ([5, 1, 1, 70, 0], [63, 64, 65, 0, 9], 2, 8, 64, 16),
    ([33, 20], [257, 100], 1, 8, 16, 12),
    ([2, 31], [300, 301], 3, 1, 32, 7),
    ([64, 1], [40, 511], 2, 4, 128, 64),
    ([9, 40], [130, 77], 1, 17, 64, 32),
    ([3, 7], [33, 200], 1, 40, 32, 128),
    ([50, 3], [20, 3], 2, 5, 80, 16),
    ([12, 30], [90, 70], 1, 4, 256, 16),
    ([21, 2], [70, 1], 2, 2, 200, 9),
]


@gpu
@BOTH
@pytest.mark.parametrize("fresh", [True, False], ids=["new", "stored"])
@pytest.mark.parametrize("shape", CHUNKS, ids=lambda s: f"{sum(s[0])}after{max(s[1])}-{s[2]}x{s[3]}x{s[4]}-{s[5]}")
def test_chunk(shape, fresh, dtype):
    counts, lengths, kv, group, dim, page = shape
    if not fresh:
        lengths = [n + c for n, c in zip(lengths, counts)]
    check_chunk(chunk_inputs(counts, lengths, kv=kv, group=group, dim=dim, page=page, dtype=dtype, fresh=fresh, sinks=fresh, seed=dim + page))


LONG_CHUNKS = [  # as many rows as the matrix-core tiles of 128 rows take
    ([130, 0, 1], [200, 5, 300], 8, 8, 64, 16),
    ([300, 35], [64, 100], 8, 4, 128, 64),
    ([70], [257], 16, 8, 32, 12),
    ([260], [40], 4, 8, 256, 7),
    ([300, 5], [90, 3], 4, 7, 80, 32),
    ([1100], [0], 1, 8, 64, 16),
    ([700], [130], 4, 3, 200, 9),
    ([40, 30], [129, 64], 3, 40, 64, 16),
    ([33, 47, 60], [1, 64, 63], 60, 1, 104, 1),
]


@gpu
@BOTH
@pytest.mark.parametrize("fresh", [True, False], ids=["new", "stored"])
@pytest.mark.parametrize("shape", LONG_CHUNKS, ids=lambda s: f"{sum(s[0])}after{max(s[1])}-{s[2]}x{s[3]}x{s[4]}-{s[5]}")
def test_long_chunk(shape, fresh, dtype):
    counts, lengths, kv, group, dim, page = shape
    if not fresh:
        lengths = [n + c for n, c in zip(lengths, counts)]
    inputs = chunk_inputs(counts, lengths, kv=kv, group=group, dim=dim, page=page, dtype=dtype, fresh=fresh, sinks=fresh, seed=dim + page)
    check_chunk(inputs)
    check_chunk(inputs, window=100, first=3)


@gpu
@BOTH
@pytest.mark.parametrize("scale", [-0.3, 0.0, 2.0])
@pytest.mark.parametrize("tokens", [9, 140])
def test_chunk_scales(tokens, scale, dtype):
    check_chunk(chunk_inputs([tokens], [50], kv=8, group=8, dim=64, page=16, dtype=dtype, seed=2), scale=scale)


@gpu
@BOTH
@pytest.mark.parametrize("window", [0, 500])
def test_long_chunk_over_a_long_cache(window, dtype):
    """Few tiles of 128 rows over many keys: a tile's keys are split over workgroups."""
    inputs = chunk_inputs([150], [2500], kv=4, group=16, dim=64, page=16, dtype=dtype, seed=3)
    call = chunk_call(**inputs, out=torch.empty_like(inputs["q"]))
    assert dtype == torch.float32 or native.library().chroma_hip_paged_chunk_attention_workspace(ctypes.byref(call)) > 0
    check_chunk(inputs, window=window, first=2)


@gpu
@BOTH
@pytest.mark.parametrize("fresh", [True, False], ids=["new", "stored"])
@pytest.mark.parametrize("window,first", [(1, 0), (2, 3), (64, 0), (128, 4), (100, 70), (5, 1000), (300, 3), (2**40, 2**40)])
def test_chunk_window_and_first_rows(window, first, fresh, dtype):
    counts, lengths = [40, 0, 1, 150, 7], [300, 4, 129, 0, 64]
    if not fresh:
        lengths = [n + c for n, c in zip(lengths, counts)]
    check_chunk(chunk_inputs(counts, lengths, kv=1, group=4, dim=32, page=16, dtype=dtype, fresh=fresh, seed=window % 97), window=window, first=first)


@gpu
@BOTH
@pytest.mark.parametrize("fresh", [True, False], ids=["new", "stored"])
@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("window,first", [(1, 1), (3, 33), (64, 64), (70, 100), (128, 130), (40, 300), (200, 5)])
def test_long_chunk_window_and_first_rows(window, first, dim, fresh, dtype):
    """Blocks of first rows alone, of both, of the window's alone."""
    counts, lengths = [30, 0, 1, 100], [400, 4, 301, 90]
    if not fresh:
        lengths = [n + c for n, c in zip(lengths, counts)]
    inputs = chunk_inputs(counts, lengths, kv=8, group=8, dim=dim, page=16, dtype=dtype, fresh=fresh, seed=window)
    inputs["table"][0, 2] = len(inputs["k_pages"])  # (a bad page: 16 rows that are not there)
    check_chunk(inputs, window=window, first=first)


@gpu
@BOTH
@pytest.mark.parametrize("counts,lengths", [([1], [4000]), ([3, 1], [2500, 0]), ([40], [1900])])
def test_chunk_of_few_tokens_over_long_caches(counts, lengths, dtype):
    """Few tiles over many rows: a tile's keys are split over workgroups."""
    inputs = chunk_inputs(counts, lengths, kv=1, group=8, dim=64, page=16, dtype=dtype, seed=3)
    call = chunk_call(**inputs, out=torch.empty_like(inputs["q"]))
    assert native.library().chroma_hip_paged_chunk_attention_workspace(ctypes.byref(call)) > 0
    check_chunk(inputs)
    check_chunk({**inputs, "sinks": None}, window=1500, first=5)


@gpu
@BOTH
def test_chunk_of_many_sequences(dtype):
    rng = np.random.default_rng(1)
    counts, lengths = rng.integers(0, 4, 150).tolist(), rng.integers(0, 40, 150).tolist()
    counts[70], counts[149] = 30, 9
    check_chunk(chunk_inputs(counts, lengths, kv=1, group=6, dim=16, page=8, dtype=dtype, seed=8))


@gpu
@BOTH
@pytest.mark.parametrize("sequences,most,group", [(65, 3, 1), (512, 2, 9), (513, 40, 16), (1300, 2, 3)])
def test_chunk_of_hundreds_of_sequences(sequences, most, group, dtype):
    """More than are counted at a time; empty ones at the ends of what a lane and a wave count; 513 fill large tiles."""
    rng = np.random.default_rng(sequences)
    counts, lengths = rng.integers(0, most + 1, sequences), rng.integers(0, 20, sequences)
    counts[[0, 7, 8, 63]], counts[-1] = 0, most
    check_chunk(chunk_inputs(counts.tolist(), lengths.tolist(), kv=1, group=group, dim=16, page=8, dtype=dtype, seed=sequences))


@gpu
@BOTH
@pytest.mark.parametrize("fresh", [True, False], ids=["new", "stored"])
@pytest.mark.parametrize("kv", [2, 80])
def test_chunk_rows_on_bad_pages_are_not_seen(kv, fresh, dtype):
    """Table entries outside the pages, lengths outside [0, longest], tokens before the first position, sequences that see
    nothing."""
    inputs = chunk_inputs([20, 6, 5, 3, 4], [100, 40, 64, 0, 90], kv=kv, group=9, dim=64, page=16, dtype=dtype, fresh=fresh, sinks=False, seed=4)
    pages = len(inputs["k_pages"])
    inputs["table"][0, 2], inputs["table"][0, 4] = -1, pages
    inputs["table"][1, :] = 2**40
    inputs["table"][2, 0] = -(2**62)
    inputs["lengths"][3], inputs["lengths"][4] = -7, 2**50  # the last one's row holds 96 entries, 6 of them rows of NaN
    inputs["k_pages"][inputs["table"][4, 5], 10:] = 0.5
    inputs["v_pages"][inputs["table"][4, 5], 10:] = -2.0
    inputs["table"] = inputs["table"][:, :6].contiguous()
    out = check_chunk(inputs)
    if not fresh:
        assert not out[20:26].any() and not out[31:34].any()


@gpu
@BOTH
def test_chunk_of_starts_out_of_order(dtype):
    inputs = chunk_inputs([4, 4, 4, 4], [10, 20, 30, 40], kv=1, group=2, dim=16, page=8, dtype=dtype, seed=6, behind=0)
    inputs["starts"] = torch.tensor([-5, 3, 2, 9, 2**40])  # sequences 0 to 3: [0, 3), none, [2, 9), [9, 16)
    inputs["starts"][2] = 3
    check_chunk(inputs)
    inputs["starts"] = torch.tensor([4, 4, 2**50, 2**60, 2**60])
    check_chunk(inputs)


@gpu
@BOTH
@pytest.mark.parametrize("where", ["new", "window", "first"])
@pytest.mark.parametrize("kv", [2, 17])
def test_chunk_values_that_are_not_finite_reach_only_who_sees_them(kv, where, dtype):
    """A value of infinity or NaN in a row that some tokens of a tile see and others do not."""
    inputs = chunk_inputs([70], [200], kv=kv, group=8, dim=64, page=16, dtype=dtype, seed=11)
    options = {} if where == "new" else {"window": 60, "first": 0 if where == "window" else 9}
    if where == "new":
        inputs["v_new"][20, 0, 3], inputs["v_new"][41, 1, 7], inputs["v_new"][41, 0, 60] = math.inf, math.nan, -math.inf
    else:
        page, row = inputs["table"][0, 160 // 16], 160 % 16
        inputs["v_pages"][page, row, 0, 5], inputs["v_pages"][page, row, 1, 33] = math.nan, -math.inf
    out = check_chunk(inputs, **options)
    assert torch.isfinite(out[:70]).any(-1).all() and not torch.isfinite(out[:70]).all()


@gpu
@BOTH
@pytest.mark.parametrize("tokens", [30, 600])
def test_chunk_of_large_and_equal_scores(tokens, dtype):
    """Scores of some hundreds (sums need the running maximum), equal ones, sinks of -inf and of the lowest value."""
    inputs = chunk_inputs([tokens, 5], [300, 65], kv=4, group=4, dim=64, page=16, dtype=dtype, seed=9, spread=6.0)
    inputs["sinks"] = torch.tensor([-math.inf, torch.finfo(dtype).min, 0.0, 300.0] * 4, dtype=dtype)
    check_chunk(inputs)
    inputs["k_pages"].nan_to_num_(0.0)
    inputs["k_pages"].fill_(0.25)
    inputs["k_new"][:-2] = 0.25
    check_chunk(inputs, scale=1.0)


@gpu
@BOTH
@pytest.mark.parametrize("tokens", [20, 150])
def test_chunk_layouts(tokens, dtype):
    """KV heads outside the rows, padded strides everywhere; what lies between out's rows stays."""
    inputs = chunk_inputs([tokens, 3], [70, 33], kv=3, group=2, dim=40, page=8, dtype=dtype, seed=3, behind=0)
    want, bound, _ = chunk_reference(**inputs)
    device, n = on_gpu(inputs), tokens + 3

    def padded(tensor, *pad):
        room = torch.full([size + p for size, p in zip(tensor.shape, pad)], math.nan, dtype=tensor.dtype, device="cuda")
        view = room[tuple(slice(0, size) for size in tensor.shape)]
        view.copy_(tensor)
        return view

    k, v = (padded(device[name].transpose(1, 2).contiguous(), 1, 0, 3, 8) for name in ("k_pages", "v_pages"))  # [P, KV, R, D]
    room = torch.full((n, 3 * 2 * 40 + 16), 7.0, dtype=dtype, device="cuda")
    out = room[:, :240].view(n, 3, 2, 40)
    q = padded(device["q"].view(n, 240), 0, 8).view(n, 3, 2, 40)
    k_new, v_new = (padded(device[name].view(n, 120), 0, 24).view(n, 3, 40) for name in ("k_new", "v_new"))
    queue_in("chroma_hip_paged_chunk_attention", chunk_call(q, k, v, device["table"], device["lengths"], device["starts"], out, k_new=k_new, v_new=v_new,
                                                            sinks=device["sinks"], heads_first=True))
    assert ((out.cpu().double() - want).abs() <= bound).all()
    assert (room[:, 240:] == 7.0).all()


@gpu
def test_chunk_offsets_past_32_bits():
    """Pages more than 2^32 elements apart."""
    inputs = chunk_inputs([20, 1], [40, 21], kv=1, group=8, dim=64, page=16, dtype=torch.bfloat16, seed=12)
    want, bound, taken = chunk_reference(**inputs)
    device = on_gpu(inputs)
    pages, stride = len(inputs["k_pages"]), (1 << 29) + 64
    room = torch.empty(pages * stride, dtype=torch.bfloat16, device="cuda")
    k = room.as_strided((pages, 16, 1, 64), (stride, 64, 64, 1))
    v = room.as_strided((pages, 16, 1, 64), (stride, 64, 64, 1), 4096)
    k.copy_(device["k_pages"])
    v.copy_(device["v_pages"])
    assert pages * stride > 1 << 32
    out = torch.empty_like(device["q"])
    queue_in("chroma_hip_paged_chunk_attention", chunk_call(**{**device, "k_pages": k, "v_pages": v}, out=out))
    assert ((out.cpu().double() - want).abs() <= bound)[taken].all()


@gpu
@BOTH
def test_chunk_in_a_graph_and_on_two_streams(dtype):
    """Two captured calls with workspaces of their own, replayed between eager work, each replay against the eager result;
    the same call twice gives the same bits."""
    first = on_gpu(chunk_inputs([3, 1], [1500, 3], kv=2, group=8, dim=64, page=16, dtype=dtype, seed=1))
    second = on_gpu(chunk_inputs([200, 8, 70], [90, 80, 70], kv=1, group=8, dim=32, page=16, dtype=dtype, seed=2))
    name = "chroma_hip_paged_chunk_attention"
    outs = [torch.zeros_like(inputs["q"]) for inputs in (first, second)]
    calls = [chunk_call(**inputs, out=out) for inputs, out in zip((first, second), outs)]
    eager, graphs, kept = [], [], []
    for call, out in zip(calls, outs):
        queue_in(name, call)
        torch.cuda.synchronize()
        eager.append(out.clone())
    for call in calls:
        need = native.library().chroma_hip_paged_chunk_attention_workspace(ctypes.byref(call))
        kept.append(torch.full((max(1, need),), 0xFF, dtype=torch.uint8, device="cuda"))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            queue_in(name, call, torch.cuda.current_stream().cuda_stream, kept[-1])
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(4):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for out, want in zip(outs, eager):
            assert torch.equal(out, want), turn
        queue_in(name, calls[turn % 2])  # the program's own eager work between the replays
        torch.cuda.synchronize()
        assert torch.equal(outs[turn % 2], eager[turn % 2])


def plain_chunk_call(**changes):
    """A valid call on addresses that are never followed."""
    fields = dict(q=1 << 20, k_pages=2 << 20, v_pages=3 << 20, k_new=4 << 20, v_new=5 << 20, sinks=6 << 20, table=7 << 20, lengths=8 << 20, starts=9 << 20,
                  out=10 << 20, tokens=5, sequences=2, kv_heads=2, group=4, dim=64, pages=10, page_rows=16, page_stride=2048, row_stride=128,
                  head_stride=64, q_stride=512, new_stride=128, out_stride=512, table_stride=4, longest=64, window=0, first=0, scale=0.125,
                  dtype=native.BFLOAT16)
    fields.update(changes)
    return native.PagedChunk(**fields)


def refused(name, call, workspace=None, size=0):
    error = ctypes.create_string_buffer(256)
    native.check(getattr(native.library(), name)(ctypes.byref(call), workspace, size, None, error, len(error)), error)


@pytest.mark.parametrize("changes,message", [
    (dict(dtype=2), "dtype"), (dict(sequences=0), "sequences"), (dict(sequences=65536), "sequences"), (dict(kv_heads=0), "KV heads"),
    (dict(group=-1), "query heads"), (dict(tokens=0), "tokens"), (dict(tokens=2**24 + 1), "tokens"), (dict(dim=0), "head dimension"),
    (dict(dim=20), "head dimension"), (dict(dim=264), "head dimension"), (dict(pages=0), "pages"), (dict(page_rows=0), "page_rows"),
    (dict(longest=-1), "longest"), (dict(longest=2**31 - 4100), "longest"), (dict(window=-1), "window"), (dict(first=-2), "first"),
    (dict(k_new=None), "k_new and v_new"), (dict(v_new=None), "k_new and v_new"), (dict(tokens=2**24, group=40), "more query rows"),
    (dict(sequences=60000, kv_heads=300), "more query rows"), (dict(table_stride=3), "table row"), (dict(longest=65), "table row"),
    (dict(q_stride=511), "stride"), (dict(out_stride=504), "stride"), (dict(new_stride=64), "stride"), (dict(row_stride=32), "stride"),
    (dict(head_stride=32), "stride"), (dict(page_stride=-2048), "stride"), (dict(q_stride=2**41), "stride"), (dict(q_stride=516), "16-byte"),
    (dict(page_stride=2052), "16-byte"), (dict(q=None), "null"), (dict(k_pages=None), "null"), (dict(v_pages=None), "null"),
    (dict(table=None), "null"), (dict(lengths=None), "null"), (dict(starts=None), "null"), (dict(out=None), "null"),
    (dict(q=(1 << 20) + 8), "16 bytes"), (dict(out=(10 << 20) + 4), "16 bytes"), (dict(k_new=(4 << 20) + 2), "16 bytes"),
    (dict(out=1 << 20), "overlaps"), (dict(out=(4 << 20) + 1024), "overlaps"), (dict(out=(8 << 20) - 4096), "overlaps"),
    (dict(out=(2 << 20) + 32768), "overlaps"), (dict(out=(3 << 20) - 16), "overlaps"), (dict(out=(6 << 20) + 16 - 16), "overlaps"),
    (dict(out=(7 << 20) + 48), "overlaps"), (dict(q_stride=2**40, out=1 << 30, tokens=2**17), "overlaps"),
    (dict(page_stride=2**40, pages=2**30, out=1 << 40), "overlaps"), (dict(tokens=2**23), "more query rows"), (dict(sequences=2**15, kv_heads=129), "more query rows"),
])
def test_chunk_refusals(changes, message):
    with pytest.raises(RuntimeError, match="paged_chunk_attention.*" + message):
        refused("chroma_hip_paged_chunk_attention", plain_chunk_call(**changes), 64 << 20, 1 << 30)


def test_chunk_workspace_refusals():
    lib = native.library()
    call = plain_chunk_call(longest=60000, table_stride=4000, pages=9000)
    need = lib.chroma_hip_paged_chunk_attention_workspace(ctypes.byref(call))
    assert need > 0
    assert lib.chroma_hip_paged_chunk_attention_workspace(ctypes.byref(plain_chunk_call(dim=20))) == 0
    for workspace, size, message in ((64 << 20, need - 1, "workspace smaller"), (None, need, "workspace smaller"), ((64 << 20) + 8, need, "16 bytes"),
                                     (1 << 20, need, "overlaps")):
        with pytest.raises(RuntimeError, match="paged_chunk_attention.*" + message):
            refused("chroma_hip_paged_chunk_attention", call, workspace, size)


# ------------------------------------------------------------------------------------------------ sampling
NEUTRAL = {"temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0}


def sample_reference(x, *, uniform, temperature=None, top_k=None, top_p=None, min_p=None):
    """[(id, logprob, nearest)] row by row in 64 bits; ``nearest``: how near the drawn place comes to the end of a token, and a
    filter's goal to a running sum (relative to the row's sum)."""
    results = []
    settings = {"temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p, "uniform": uniform}
    for r, row in enumerate(x.float().numpy().astype(np.float64)):
        one = {name: NEUTRAL.get(name) if values is None else values[r].item() for name, values in settings.items()}
        if np.isnan(row).any():
            results.append((int(np.flatnonzero(np.isnan(row))[0]), math.nan, 1.0))
            continue
        top = row.max()
        if top == -math.inf:
            results.append((-1, -math.inf, 1.0))
            continue
        if not one["temperature"] > 0:
            results.append((int(row.argmax()), 0.0, 1.0))
            continue
        order = np.lexsort((np.arange(len(row)), -row))
        with np.errstate(invalid="ignore"):
            depth = np.where(row == top, 0.0, (top - row) / one["temperature"])[order]
        depth = np.where(np.isnan(depth), math.inf, depth)
        weights = np.exp(-depth)
        kept, nearest = len(row), 1.0
        if 0 < one["top_k"] < len(row):
            kept = int(one["top_k"])
        if one["top_p"] < 1:
            sums = np.cumsum(weights)
            goal = one["top_p"] * sums[kept - 1]
            nearest = min(nearest, np.abs(sums - goal).min() / sums[-1])
            kept = min(kept, int((sums < goal).sum()) + 1)
        if one["min_p"] > 0:
            kept = max(1, min(kept, int((weights >= one["min_p"]).sum())))
        weights = weights[:kept]
        sums = np.cumsum(weights)
        u = one["uniform"]
        u = 0.0 if not u > 0 else min(u, float(np.float32(1) - np.float32(2.0**-24)))
        chosen = min(int((sums <= u * sums[-1]).sum()), kept - 1)
        while weights[chosen] == 0:
            chosen -= 1
        nearest = min(nearest, np.abs(sums - u * sums[-1])[: kept - 1].min() / sums[-1] if kept > 1 else 1.0)
        results.append((int(order[chosen]), -depth[chosen] - math.log(sums[-1]), nearest))
    return results


def sample_call(x, ids, logprobs, *, uniform, temperature=None, top_k=None, top_p=None, min_p=None):
    rows, width = x.shape
    return native.Sample(x=pointer(x), rows=rows, width=width, x_stride=x.stride(0), temperature=pointer(temperature), top_k=pointer(top_k),
                         top_p=pointer(top_p), min_p=pointer(min_p), uniform=pointer(uniform), ids=pointer(ids), logprobs=pointer(logprobs),
                         dtype=DTYPES[x.dtype])


def sampled(x, **settings):
    ids = torch.full((len(x),), -99, dtype=torch.int64, device="cuda")
    logprobs = torch.full((len(x),), 55.0, device="cuda")
    device = {name: None if values is None else values.cuda() for name, values in settings.items()}
    x = x.cuda() if x.device.type == "cpu" else x
    queue_in("chroma_hip_rows_sample", sample_call(x, ids, logprobs, **device))
    return ids.cpu(), logprobs.cpu()


def check_sample(x, **settings):
    """Every id must be the reference's, but where the place lies within 1e-9 of a border: sums of 2^19 units of 2^-44, each
    half a unit off, and the reference's own 64-bit sums."""
    want = sample_reference(x.cpu(), **settings)
    ids, logprobs = sampled(x, **settings)
    for r, (token, logprob, nearest) in enumerate(want):
        if 0 < nearest < 1e-9:
            continue
        assert int(ids[r]) == token, (r, nearest)
        # one rounding of the value, and 2^19 units of 2^-45 of the sum
        np.testing.assert_allclose(float(logprobs[r]), logprob, rtol=2.0**-24 + 1e-12, atol=2.0**-24 + 2e-8 * 2.0**-3, err_msg=str(r))
    return ids, logprobs


def row_settings(rows, seed=0):
    g = torch.Generator().manual_seed(seed)

    def pick(*values):
        return torch.tensor(values)[torch.randint(0, len(values), (rows,), generator=g)]

    return {"uniform": torch.rand(rows, generator=g), "temperature": pick(0.0, 0.1, 0.7, 1.0, 1.0, 2.5, 30.0),
            "top_k": pick(0, 0, 1, 2, 5, 40, 1000, 2**40, -3), "top_p": pick(1.0, 1.0, 0.9, 0.5, 0.99, 0.0, 1e-30), "min_p": pick(0.0, 0.0, 0.05, 1e-4, 0.9)}


@gpu
@BOTH
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 2), (40, 7), (64, 63), (64, 65), (90, 1000), (33, 4099), (20, 32000), (12, 201088)])
def test_sample(rows, width, dtype):
    x = (torch.randn(rows, width, generator=torch.Generator().manual_seed(width)) * 3).to(dtype)
    settings = row_settings(rows, seed=rows)
    check_sample(x, **settings)
    check_sample(x, uniform=settings["uniform"])
    for name in ("temperature", "top_k", "top_p", "min_p"):
        check_sample(x, uniform=settings["uniform"], **{name: settings[name]})


@gpu
@BOTH
@pytest.mark.parametrize("rows,width", [(1, 16384), (2, 70001), (70, 16390), (300, 9001), (300, 4096), (5, 4097)])
@pytest.mark.parametrize("spread", [0.001, 2.0, 40.0])
def test_sample_cut_into_spans_or_not(rows, width, spread, dtype):
    """Few rows are cut into spans; logits that lie close together or far apart."""
    x = (torch.randn(rows, width, generator=torch.Generator().manual_seed(width)) * spread).to(dtype)
    settings = row_settings(rows, seed=rows + 1)
    check_sample(x, **settings)
    check_sample(x, uniform=settings["uniform"], top_p=settings["top_p"], min_p=settings["min_p"])


@gpu
@BOTH
@pytest.mark.parametrize("rows,width", [(3, 40000), (200, 12000)])
def test_sample_of_rows_that_no_list_holds(rows, width, dtype):
    """Equal values, few distinct ones, a large top_k, high temperatures: a bucket holds more than a list."""
    g = torch.Generator().manual_seed(width)
    x = torch.randint(-3, 4, (rows, width), generator=g).to(dtype)
    x[0] = 0.25
    settings = row_settings(rows, seed=7)
    check_sample(x, **settings)
    check_sample(x, **{**settings, "top_k": torch.full((rows,), width - 5)})
    x = torch.randn(rows, width, generator=g).to(dtype)
    check_sample(x, uniform=settings["uniform"], top_k=torch.full((rows,), 3000))
    check_sample(x, uniform=settings["uniform"], temperature=torch.full((rows,), 500.0), top_p=torch.full((rows,), 0.7))


@gpu
@BOTH
def test_sample_of_ties_and_equal_rows(dtype):
    """Few distinct values, rows all equal, both zeros: ties go by id, and cuts fall among them."""
    g = torch.Generator().manual_seed(3)
    x = torch.randint(-2, 3, (60, 5000), generator=g).to(dtype)
    x[:20] = 1.5
    x[20:40] *= 0.0  # zeros of both signs
    check_sample(x, **row_settings(60, seed=5))
    # 5000 equal tokens: a place of u * 5000 names its token
    u = torch.arange(60) / 60 + 1e-3
    ids, _ = check_sample(x, uniform=u)
    assert ids[:40].tolist() == [int(float(v) * 5000) for v in u[:40]]


@gpu
@BOTH
def test_sample_of_infinite_and_missing_logits(dtype):
    x = torch.randn(12, 700, generator=torch.Generator().manual_seed(2)).to(dtype)
    x[0] = -math.inf
    x[1, 5:] = -math.inf
    x[2, 100], x[2, 600] = math.inf, math.inf
    x[3, 44], x[3, 45], x[3, 2] = math.nan, math.nan, math.inf
    x[4, :] = torch.finfo(dtype).min
    x[5, :] = torch.finfo(dtype).min
    x[5, 77] = torch.finfo(dtype).max
    x[6, 1:] = -math.inf
    x[7, ::2] = -math.inf
    x[8, 300] = math.nan
    settings = {"uniform": torch.tensor([0.5, 0.99, 0.7, 0.1, 0.5, 0.9, 0.999, 0.4, 0.3, 0.2, 0.6, 0.8]), "temperature": torch.full((12,), 0.8)}
    ids, logprobs = check_sample(x, **settings)
    assert int(ids[0]) == -1 and int(ids[2]) == 600 and int(ids[3]) == 44 and int(ids[5]) == 77
    check_sample(x, **settings, top_k=torch.full((12,), 600), top_p=torch.full((12,), 0.9), min_p=torch.full((12,), 0.001))
    check_sample(x, **{**settings, "temperature": torch.zeros(12)})
    check_sample(x, **{**settings, "temperature": torch.full((12,), math.inf)})
    check_sample(x, **{**settings, "temperature": torch.full((12,), 1e-30)})


@gpu
@BOTH
def test_sample_of_settings_at_their_ends(dtype):
    """Random numbers outside [0, 1), NaN settings, filters of 0, of 1 and beyond."""
    nan, inf = math.nan, math.inf
    x = (torch.randn(1, 900, generator=torch.Generator().manual_seed(4)) * 2).to(dtype).expand(12, 900).contiguous()
    uniform = torch.tensor([0.0, -1.0, 1.0, 7.0, nan, 1.0 - 2.0**-24, 1e-45, 1e-10, inf, -inf, 0.5, 0.25])
    half = torch.full((12,), 0.5)
    ids, _ = check_sample(x, uniform=uniform)
    order = torch.sort(x[0].float(), descending=True, stable=True)[1]
    assert ids[0] == ids[1] == ids[4] == ids[6] == ids[9] == order[0] and ids[2] == ids[3] == ids[8] == ids[5] == order[-1]
    check_sample(x, uniform=half, top_p=torch.tensor([0.0, -1.0, 1.0, 7.0, 1.0, 1.0 - 2.0**-24, 1e-45, 1e-10, inf, -inf, 0.5, 0.25]))
    check_sample(x, uniform=half, min_p=torch.tensor([0.0, -1.0, 1.0, 7.0, 0.0, 1.0 - 2.0**-24, 1e-45, 1e-10, inf, -inf, 0.5, 0.25]))
    plain, greedy = check_sample(x, uniform=half)[0], check_sample(x, uniform=half, temperature=torch.zeros(12))[0]
    some = torch.full((12,), nan)
    assert torch.equal(sampled(x, uniform=half, top_p=some)[0], plain) and torch.equal(sampled(x, uniform=half, min_p=some)[0], plain)
    assert torch.equal(sampled(x, uniform=half, temperature=some)[0], greedy)


@gpu
@BOTH
@pytest.mark.parametrize("width", [900, 40000])
@pytest.mark.parametrize("spread", [1e-6, 1e-3, 0.05, 1.0])
def test_sample_of_flat_rows(spread, width, dtype):
    """Whole rows within a small factor, or nothing: their own depths are what the buckets are spread over."""
    x = torch.randn(6, width, generator=torch.Generator().manual_seed(3)) * spread
    x[1, ::7] = -math.inf
    x[2] = 30 + x[2]
    x[3, 1:] = -math.inf
    x[4, 5] = spread * 9
    x = x.to(dtype)
    uniform = torch.rand(6, generator=torch.Generator().manual_seed(1))
    for filters in ({}, {"min_p": torch.tensor([0.999, 0.9, 1.0, 0.5, 1 - 2.0**-20, 1 - 1e-6])}, {"top_p": torch.full((6,), 0.4)}, {"top_k": torch.full((6,), 400)},
                    {"temperature": torch.full((6,), 40.0), "top_k": torch.tensor([0, 5, 1000, 0, 70, 0]), "top_p": torch.full((6,), 0.9), "min_p": torch.full((6,), 0.97)}):
        check_sample(x, uniform=uniform, **filters)


@gpu
@BOTH
@pytest.mark.parametrize("width", [900, 40000])
def test_sample_at_the_least_temperatures(width, dtype):
    """Temperatures whose inverse is no float, with logits that differ by as little, and with others."""
    temperature = torch.tensor([1e-36, 3e-37, 1e-37, 1e-38, 1e-40, 1e-45, 1e-45, 1e-38])
    x = torch.randn(8, width, generator=torch.Generator().manual_seed(9))
    x = torch.cat((x[:6] * temperature[:6, None].clamp(min=1e-38), x[6:])).to(dtype)
    uniform = torch.rand(8, generator=torch.Generator().manual_seed(2))
    for filters in ({}, {"top_k": torch.full((8,), 50)}, {"top_p": torch.full((8,), 0.9)}, {"min_p": torch.full((8,), 0.1)}):
        check_sample(x, uniform=uniform, temperature=temperature, **filters)


@gpu
@BOTH
def test_sample_layouts(dtype):
    """Rows apart and off any alignment, no logprobs."""
    room = torch.full((9, 1333), math.nan, dtype=dtype)
    x = room[:, 3:1004]
    x.copy_(torch.randn(9, 1001, generator=torch.Generator().manual_seed(6)))
    settings = row_settings(9, seed=2)
    want, _ = check_sample(x, **settings)
    device = {name: values.cuda() for name, values in settings.items()}
    ids, x = torch.full((9,), -9, dtype=torch.int64, device="cuda"), room.cuda()[:, 3:1004]
    assert x.stride(0) == 1333
    queue_in("chroma_hip_rows_sample", sample_call(x, ids, None, **device))
    assert torch.equal(ids.cpu(), want)


@gpu
@BOTH
def test_sample_in_a_graph_and_on_two_streams(dtype):
    x = [(torch.randn(rows, 30011, generator=torch.Generator().manual_seed(rows)) * 3).to(dtype) for rows in (5, 40)]
    settings = [row_settings(rows, seed=9) for rows in (5, 40)]
    want = [check_sample(one, **setting) for one, setting in zip(x, settings)]
    graphs, kept = [], []
    for one, setting in zip(x, settings):
        device, one = {name: values.cuda() for name, values in setting.items()}, one.cuda()
        ids, logprobs = torch.zeros(len(one), dtype=torch.int64, device="cuda"), torch.zeros(len(one), device="cuda")
        call = sample_call(one, ids, logprobs, **device)
        workspace = queue_in("chroma_hip_rows_sample", call)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            queue_in("chroma_hip_rows_sample", call, torch.cuda.current_stream().cuda_stream, workspace)
        graphs.append(graph)
        kept.append((one, device, ids, logprobs, workspace))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(4):
        for _, _, ids, logprobs, _ in kept:
            ids.fill_(-5)
            logprobs.fill_(9.0)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for (_, _, ids, logprobs, _), (want_ids, want_logprobs) in zip(kept, want):
            assert torch.equal(ids.cpu(), want_ids) and torch.equal(logprobs.cpu(), want_logprobs), turn
        assert torch.equal(sampled(x[turn % 2], **settings[turn % 2])[0], want[turn % 2][0])


def plain_sample_call(**changes):
    fields = dict(x=1 << 20, rows=2, width=100, x_stride=100, temperature=2 << 20, top_k=3 << 20, top_p=4 << 20, min_p=5 << 20, uniform=6 << 20,
                  ids=7 << 20, logprobs=8 << 20, dtype=native.FLOAT32)
    fields.update(changes)
    return native.Sample(**fields)


@pytest.mark.parametrize("changes,message", [
    (dict(dtype=2), "dtype"), (dict(rows=0), "rows"), (dict(rows=65536), "rows"), (dict(width=0), "logits"), (dict(width=2**19 + 1, x_stride=2**20), "logits"),
    (dict(x_stride=99), "x_stride"), (dict(x_stride=2**41), "x_stride"), (dict(x=None), "null"), (dict(uniform=None), "null"), (dict(ids=None), "null"),
    (dict(x=(1 << 20) + 2), "own size"), (dict(ids=1 << 20), "overlap"), (dict(logprobs=6 << 20), "overlap"), (dict(logprobs=(7 << 20) + 12), "overlap"),
    (dict(ids=(3 << 20) - 8), "overlap"),
])
def test_sample_refusals(changes, message):
    with pytest.raises(RuntimeError, match="rows_sample.*" + message):
        refused("chroma_hip_rows_sample", plain_sample_call(**changes), 64 << 20, 1 << 30)


@pytest.mark.parametrize("name,workspace", [("chroma_hip_paged_plan", False), ("chroma_hip_cache_store", False),
                                            ("chroma_hip_paged_chunk_attention", True), ("chroma_hip_rows_sample", True)])
def test_null_calls_are_refused(name, workspace):
    error = ctypes.create_string_buffer(256)
    status = getattr(native.library(), name)(None, *([None, 0] if workspace else []), None, error, len(error))
    assert status == native.RUNTIME_ERROR and b"null call" in error.value
