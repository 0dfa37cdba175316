"""The operators of batched decoding through the C ABI (paged attention, cache row moves, logit adjustments) against
plain 64-bit implementations, and their refusals. Refusals are decided on the host, so they run without a GPU."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

from chroma_amd._src import native

gpu = pytest.mark.gpu
DTYPES = {torch.float32: native.FLOAT32, torch.bfloat16: native.BFLOAT16}
HALF = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8}  # half a step relative to a value


def checked(status, error):
    native.check(status, error)


def pointer(tensor):
    return None if tensor is None else tensor.data_ptr()


# ------------------------------------------------------------------------------------------------ paged attention
def attention_call(q, k_pages, v_pages, table, lengths, out, *, k_new=None, v_new=None, sinks=None, longest=None, window=0, first=0,
                   scale=None, heads_first=False):
    """The call for tensors: q and out [B, KV, G, D], pages [P, R, KV, D] (or [P, KV, R, D])."""
    n, kv, group, dim = q.shape
    rows = k_pages.shape[2 if heads_first else 1]
    row_stride, head_stride = k_pages.stride()[2 if heads_first else 1], k_pages.stride()[1 if heads_first else 2]
    return native.PagedAttention(
        q=pointer(q), k_pages=pointer(k_pages), v_pages=pointer(v_pages), k_new=pointer(k_new), v_new=pointer(v_new), sinks=pointer(sinks),
        table=pointer(table), lengths=pointer(lengths), out=pointer(out), sequences=n, kv_heads=kv, group=group, dim=dim,
        pages=k_pages.shape[0], page_rows=rows, page_stride=k_pages.stride()[0], row_stride=row_stride, head_stride=head_stride,
        q_stride=q.stride()[0], new_stride=0 if k_new is None else k_new.stride()[0], out_stride=out.stride()[0],
        table_stride=table.stride()[0], longest=table.shape[1] * rows if longest is None else longest, window=window, first=first,
        scale=dim**-0.5 if scale is None else scale, dtype=DTYPES[q.dtype])


def attend(call, stream=None, workspace=None):
    lib, error = native.library(), ctypes.create_string_buffer(256)
    need = lib.chroma_hip_paged_attention_workspace(ctypes.byref(call))
    if workspace is None:
        workspace = torch.full((max(1, need),), 0xAB, dtype=torch.uint8, device="cuda")
    checked(lib.chroma_hip_paged_attention(ctypes.byref(call), workspace.data_ptr(), workspace.numel(), stream, error, len(error)), error)
    return workspace


def attention_reference(q, k_pages, v_pages, table, lengths, *, k_new=None, v_new=None, sinks=None, longest=None, window=0, first=0,
                        scale=None):
    """(result in 64 bits, bound of a float evaluation rounded once to q's type) on the CPU; pages [P, R, KV, D].

    The bound: a score's products and sum, (D + 3) roundings of at most sum |q k|; a weight's exponential, 1.2e-7 + 6e-8 |x|
    relative (device.h); a sum of n weighted values in any order, n roundings of at most sum p |v|; for bfloat16 also the
    weight held as two bfloat16 halves, 2^-16; and half a step of the result."""
    n, kv, group, dim = q.shape
    dtype, rows = q.dtype, k_pages.shape[1]
    longest = table.shape[1] * rows if longest is None else longest
    scale = dim**-0.5 if scale is None else scale
    result, bound = torch.zeros(n, kv, group, dim, dtype=torch.float64), torch.zeros(n, kv, group, 1, dtype=torch.float64)
    for b in range(n):
        length = min(max(int(lengths[b]), 0), longest)
        position = length if k_new is not None else length - 1
        k, v = [], []
        for j in range(length):
            page = int(table[b, j // rows])
            if 0 <= page < k_pages.shape[0] and (not window or j > position - window or j < first):
                k.append(k_pages[page, j % rows])
                v.append(v_pages[page, j % rows])
        if k_new is not None:
            k.append(k_new[b])
            v.append(v_new[b])
        if not k:
            continue
        k, v = torch.stack(k).double(), torch.stack(v).double()  # [S, KV, D]
        for h in range(kv):
            products = q[b, h].double()[:, None, :] * k[None, :, h]
            s = products.sum(-1) * scale
            off = (dim + 3) * 2.0**-24 * products.abs().sum(-1).amax(-1) * abs(scale)
            extra = sinks.double().view(kv, group)[h][:, None] if sinks is not None else torch.full((group, 1), -math.inf, dtype=torch.float64)
            joined = torch.cat([s, extra], 1)
            p = torch.softmax(joined, 1)[:, : len(k)]
            result[b, h] = p @ v[:, h]
            reach = (joined.amax(1, keepdim=True) - joined)[torch.isfinite(joined)].amax().clamp(max=90.0)
            relative = 2 * off + 2 * (1.2e-7 + 6e-8 * float(reach)) + 2 * (len(k) + 8) * 2.0**-24
            if dtype == torch.bfloat16:
                relative = relative + 2.0**-16
            bound[b, h, :, 0] = relative * v[:, h].abs().amax()
    return result, bound + HALF[dtype] * result.abs() + 1e-37


def paged_inputs(lengths, *, kv, group, dim, page, dtype, fresh=True, sinks=True, seed=0, spread=1.0, spare=3):
    """CPU tensors; pages in random order, rows behind a sequence's last and unused pages hold NaN and infinities."""
    g = torch.Generator().manual_seed(seed)
    span = max(1, -(-max(lengths) // page))
    used = [-(-max(0, n) // page) for n in lengths]
    pages = sum(used) + spare
    order = torch.randperm(pages, generator=g)
    table = torch.full((len(lengths), span), -1, dtype=torch.int64)

    def values(*shape):
        return (torch.randn(*shape, generator=g) * spread).to(dtype)

    k = torch.full((pages, page, kv, dim), math.nan, dtype=dtype)
    v = torch.full((pages, page, kv, dim), math.inf, dtype=dtype)
    taken = 0
    for b, n in enumerate(lengths):
        for i in range(used[b]):
            table[b, i] = order[taken]
            rows = min(page, n - i * page)
            k[order[taken], :rows], v[order[taken], :rows] = values(rows, kv, dim), values(rows, kv, dim)
            taken += 1
    return {"q": values(len(lengths), kv, group, dim), "k_pages": k, "v_pages": v, "table": table,
            "lengths": torch.tensor(lengths, dtype=torch.int64), "k_new": values(len(lengths), kv, dim) if fresh else None,
            "v_new": values(len(lengths), kv, dim) if fresh else None, "sinks": values(kv * group) if sinks else None}


def on_gpu(inputs):
    return {name: None if value is None else value.cuda() for name, value in inputs.items()}


def check_attention(inputs, **options):
    want, bound = attention_reference(**inputs, **options)
    device = on_gpu(inputs)
    out = torch.full(device["q"].shape, math.nan, dtype=device["q"].dtype, device="cuda")
    attend(attention_call(**device, out=out, **options))
    got = out.cpu().double()
    assert torch.isfinite(got).all()
    excess = ((got - want).abs() - bound).amax()
    assert excess <= 0, f"off by {float((got - want).abs().amax())}, {float(excess)} more than the bound"
    return out


SHAPES = [  # (lengths, kv, group, dim, page)
    ([1], 1, 1, 8, 1),
    ([0, 1, 2, 15, 16, 17], 2, 3, 16, 16),
    ([63, 64, 65, 128, 129, 0], 2, 8, 64, 16),
    ([257, 5, 1000], 1, 8, 16, 12),
    ([300, 301], 3, 1, 32, 7),
    ([511, 40, 1], 2, 16, 128, 64),
    ([130, 77], 2, 17, 64, 32),
    ([33, 400], 1, 40, 32, 128),
    ([200, 3], 2, 5, 80, 16),
    ([90, 250], 1, 4, 256, 16),
    ([70, 1], 2, 2, 200, 9),
    ([1500], 8, 8, 64, 16),
]


LONG_SHAPES = [  # more key blocks than one workgroup takes; a wave knows the lengths of 64 sequences from one load
    ([4000], 1, 3, 64, 16),
    ([2100, 1900], 1, 8, 8, 5),
    ([9000, 0, 1], 2, 2, 256, 64),
    ([1, 2500, 0, 700] * 18, 2, 4, 32, 16),
    ([0] * 63 + [3200, 3000, 0, 1, 40] + [10] * 60 + [2000, 0], 1, 17, 16, 12),
]


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("window,first", [(0, 0), (1800, 3)])
@pytest.mark.parametrize("shape", LONG_SHAPES, ids=lambda s: f"{len(s[0])}x{max(s[0])}-{s[1]}x{s[2]}x{s[3]}-{s[4]}")
def test_paged_attention_of_long_sequences(shape, window, first, dtype):
    lengths, kv, group, dim, page = shape
    inputs = paged_inputs(lengths, kv=kv, group=group, dim=dim, page=page, dtype=dtype, fresh=not window, sinks=bool(window), seed=dim)
    call = attention_call(**inputs, out=torch.empty_like(inputs["q"]), window=window, first=first)
    assert native.library().chroma_hip_paged_attention_workspace(ctypes.byref(call)) > 0
    check_attention(inputs, window=window, first=first)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("fresh", [True, False], ids=["new", "stored"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{len(s[0])}x{max(s[0])}-{s[1]}x{s[2]}x{s[3]}-{s[4]}")
def test_paged_attention(shape, fresh, dtype):
    lengths, kv, group, dim, page = shape
    check_attention(paged_inputs(lengths, kv=kv, group=group, dim=dim, page=page, dtype=dtype, fresh=fresh, sinks=fresh, seed=dim + page))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("fresh", [True, False], ids=["new", "stored"])
@pytest.mark.parametrize("window,first", [(1, 0), (2, 0), (64, 0), (128, 4), (100, 70), (5, 1000), (2000, 3), (2**40, 2**40)])
def test_paged_attention_window_and_first_rows(window, first, fresh, dtype):
    inputs = paged_inputs([0, 1, 5, 64, 128, 129, 700], kv=2, group=4, dim=32, page=16, dtype=dtype, fresh=fresh, seed=window % 97)
    check_attention(inputs, window=window, first=first)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("fresh", [True, False], ids=["new", "stored"])
def test_paged_attention_rows_on_bad_pages_are_not_seen(fresh, dtype):
    """Table entries outside the pages, lengths outside [0, longest], a sequence that sees nothing."""
    inputs = paged_inputs([100, 40, 64, 0, 90], kv=2, group=3, dim=64, page=16, dtype=dtype, fresh=fresh, sinks=False, seed=4)
    pages = len(inputs["k_pages"])
    inputs["table"][0, 2], inputs["table"][0, 4] = -1, pages
    inputs["table"][1, :] = 2**40
    inputs["table"][2, 0] = -(2**62)
    inputs["lengths"][3], inputs["lengths"][4] = -7, 2**50  # the last one's row holds 96 entries, 6 of them rows of NaN
    inputs["k_pages"][inputs["table"][4, 5], 10:] = 0.5
    inputs["v_pages"][inputs["table"][4, 5], 10:] = -2.0
    inputs["table"] = inputs["table"][:, :6].contiguous()
    out = check_attention(inputs)
    if not fresh:
        assert not out[1].any() and not out[3].any()


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_paged_attention_of_large_and_equal_scores(dtype):
    """Scores of some hundreds (sums need the running maximum), equal ones, and a sink of -inf and one of the lowest value."""
    inputs = paged_inputs([700, 65], kv=1, group=4, dim=64, page=16, dtype=dtype, seed=9, spread=6.0)
    inputs["sinks"] = torch.tensor([-math.inf, torch.finfo(dtype).min, 0.0, 300.0], dtype=dtype)
    check_attention(inputs)
    inputs["k_pages"].nan_to_num_(0.0)
    inputs["k_pages"].fill_(0.25)
    check_attention(inputs, scale=1.0)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_paged_attention_layouts(dtype):
    """KV heads outside the rows, padded strides everywhere; what lies between out's rows stays."""
    inputs = paged_inputs([70, 33], kv=3, group=2, dim=40, page=8, dtype=dtype, seed=3)
    want, bound = attention_reference(**inputs)
    device = on_gpu(inputs)

    def padded(tensor, *pad):
        room = torch.full([n + p for n, p in zip(tensor.shape, pad)], math.nan, dtype=tensor.dtype, device="cuda")
        view = room[tuple(slice(0, n) for n in tensor.shape)]
        view.copy_(tensor)
        return view

    # [P, KV, R, D] with longer rows, longer pages
    k, v = (padded(device[name].transpose(1, 2).contiguous(), 1, 0, 3, 8) for name in ("k_pages", "v_pages"))
    room = torch.full((2, 3 * 2 * 40 + 16), 7.0, dtype=dtype, device="cuda")
    out = room[:, :240].view(2, 3, 2, 40)
    q = torch.full((2, 3 * 2 * 40 + 8), math.nan, dtype=dtype, device="cuda")[:, :240].view(2, 3, 2, 40)
    q.copy_(device["q"])
    k_new, v_new = (torch.full((2, 3 * 40 + 24), math.nan, dtype=dtype, device="cuda")[:, :120].view(2, 3, 40) for _ in range(2))
    k_new.copy_(device["k_new"])
    v_new.copy_(device["v_new"])
    table = padded(device["table"].double(), 0, 0).long()
    table = torch.cat([table, torch.full((2, 5), 10**9, device="cuda", dtype=torch.int64)], 1)[:, : table.shape[1]]
    attend(attention_call(q, k[: len(inputs["k_pages"])], v[: len(inputs["k_pages"])], table, device["lengths"], out, k_new=k_new, v_new=v_new,
                          sinks=device["sinks"], heads_first=True))
    assert ((out.cpu().double() - want).abs() <= bound).all()
    assert (room[:, 240:] == 7.0).all()


@gpu
def test_paged_attention_offsets_past_32_bits():
    """Pages more than 2^32 elements apart."""
    inputs = paged_inputs([40, 21], kv=1, group=8, dim=64, page=16, dtype=torch.bfloat16, seed=12, spare=0)
    want, bound = attention_reference(**inputs)
    device = on_gpu(inputs)
    pages, stride = len(inputs["k_pages"]), (1 << 30) + 64
    room = torch.empty(pages * stride, dtype=torch.bfloat16, device="cuda")
    k = room.as_strided((pages, 16, 1, 64), (stride, 64, 64, 1))
    v = room.as_strided((pages, 16, 1, 64), (stride, 64, 64, 1), 4096)
    k.copy_(device["k_pages"])
    v.copy_(device["v_pages"])
    assert pages * stride > 1 << 32
    out = torch.empty_like(device["q"])
    attend(attention_call(device["q"], k, v, device["table"], device["lengths"], out, k_new=device["k_new"], v_new=device["v_new"],
                          sinks=device["sinks"]))
    assert ((out.cpu().double() - want).abs() <= bound).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_paged_attention_in_a_graph_and_on_two_streams(dtype):
    """Two captured calls with workspaces of their own, replayed between eager work, each replay against the eager result;
    the same call twice gives the same bits."""
    first = on_gpu(paged_inputs([1200, 3], kv=2, group=8, dim=64, page=16, dtype=dtype, seed=1))
    second = on_gpu(paged_inputs([900, 800, 70], kv=1, group=8, dim=32, page=16, dtype=dtype, seed=2))
    outs = [torch.empty_like(inputs["q"]) for inputs in (first, second)]
    calls = [attention_call(**inputs, out=out) for inputs, out in zip((first, second), outs)]
    eager = []
    for call, out in zip(calls, outs):
        attend(call)
        torch.cuda.synchronize()
        eager.append(out.clone())
    graphs, kept = [], []
    for call in calls:
        need = native.library().chroma_hip_paged_attention_workspace(ctypes.byref(call))
        kept.append(torch.full((max(1, need),), 0xFF, dtype=torch.uint8, device="cuda"))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            attend(call, torch.cuda.current_stream().cuda_stream, kept[-1])
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(4):
        for out in outs:
            out.fill_(math.nan)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for out, want in zip(outs, eager):
            assert torch.equal(out, want), turn
        attend(calls[turn % 2])  # the program's own eager work between the replays
        torch.cuda.synchronize()
        assert torch.equal(outs[turn % 2], eager[turn % 2])


def plain_attention_call(**changes):
    """A valid call on addresses that are never followed."""
    fields = dict(q=4096, k_pages=8192, v_pages=12288, k_new=16384, v_new=20480, sinks=24576, table=28672, lengths=32768, out=36864,
                  sequences=2, kv_heads=2, group=4, dim=64, pages=10, page_rows=16, page_stride=2048, row_stride=128, head_stride=64,
                  q_stride=512, new_stride=128, out_stride=512, table_stride=4, longest=64, window=0, first=0, scale=0.125,
                  dtype=native.BFLOAT16)
    fields.update(changes)
    return native.PagedAttention(**fields)


@pytest.mark.parametrize("changes,message", [
    (dict(dtype=2), "dtype"), (dict(sequences=0), "sequences"), (dict(sequences=65536), "sequences"), (dict(kv_heads=0), "KV heads"),
    (dict(group=-1), "query heads"), (dict(dim=0), "head dimension"), (dict(dim=20), "head dimension"), (dict(dim=264), "head dimension"),
    (dict(pages=0), "pages"), (dict(page_rows=0), "page_rows"), (dict(longest=-1), "longest"), (dict(longest=2**31), "longest"),
    (dict(window=-1), "window"), (dict(first=-2), "first"), (dict(k_new=None), "k_new and v_new"), (dict(v_new=None), "k_new and v_new"),
    (dict(sequences=60000, kv_heads=300), "more query heads"), (dict(sequences=40000, longest=2**21, table_stride=2**17), "more sequences"),
    (dict(table_stride=3), "table row"), (dict(longest=65), "table row"), (dict(q_stride=511), "stride"), (dict(out_stride=504), "stride"),
    (dict(new_stride=64), "stride"), (dict(row_stride=32), "stride"), (dict(head_stride=32), "stride"), (dict(page_stride=-2048), "stride"),
    (dict(q_stride=516), "16-byte"), (dict(page_stride=2052), "16-byte"), (dict(q=None), "null"), (dict(k_pages=None), "null"),
    (dict(v_pages=None), "null"), (dict(table=None), "null"), (dict(lengths=None), "null"), (dict(out=None), "null"),
    (dict(q=4104), "16 bytes"), (dict(v_pages=12290), "16 bytes"), (dict(v_new=20488), "16 bytes"),
])
def test_paged_attention_refusals(changes, message):
    error = ctypes.create_string_buffer(256)
    call = plain_attention_call(**changes)
    status = native.library().chroma_hip_paged_attention(ctypes.byref(call), None, 0, None, error, len(error))
    assert status == native.RUNTIME_ERROR and error.value.decode().startswith("paged_attention: ") and message in error.value.decode()


def test_paged_attention_refuses_no_call_and_a_short_workspace():
    lib, error = native.library(), ctypes.create_string_buffer(256)
    assert lib.chroma_hip_paged_attention(None, None, 0, None, error, len(error)) == native.RUNTIME_ERROR
    assert lib.chroma_hip_paged_attention_workspace(ctypes.byref(plain_attention_call(dim=20))) == 0
    call = plain_attention_call(sequences=1, longest=100000, table_stride=6250)
    need = lib.chroma_hip_paged_attention_workspace(ctypes.byref(call))
    if need:
        for workspace, size in ((None, need), (65536, need - 1)):
            assert lib.chroma_hip_paged_attention(ctypes.byref(call), workspace, size, None, error, len(error)) == native.RUNTIME_ERROR
            assert b"workspace" in error.value


# ------------------------------------------------------------------------------------------------ cache rows
def cache_of(keys, values):
    return native.CacheRows(keys=keys.data_ptr(), values=values.data_ptr(), rows=keys.shape[1], layer_pitch=keys.stride()[0] * keys.element_size())


def move(to, source, moves, layers, row_bytes, stream=None):
    lib, error = native.library(), ctypes.create_string_buffer(256)
    moves = np.ascontiguousarray(moves, dtype=np.int64).reshape(-1, 3)
    checked(lib.chroma_hip_cache_move(ctypes.byref(to), ctypes.byref(source), layers, row_bytes, moves.ctypes.data, len(moves), stream,
                                      error, len(error)), error)


def moved(target, source, moves):
    """The rule on host arrays [layers, rows, bytes]."""
    result = target.clone()
    for first, to, rows in moves:
        result[:, to : to + rows] = source[:, first : first + rows]
    return result


def disjoint_moves(rng, rows, count, most):
    """Moves inside a cache of ``rows`` rows whose targets and sources are runs of their own."""
    slots = rng.permutation(rows // most)[: 2 * count] * most
    sizes = rng.integers(0, most + 1, count)
    return [(int(slots[2 * i]), int(slots[2 * i + 1]), int(sizes[i])) for i in range(count)]


@gpu
@pytest.mark.parametrize("layers,row_bytes,rows,count,most", [(1, 1, 40, 3, 5), (3, 16, 200, 10, 8), (2, 1000, 100, 7, 7), (5, 128, 3000, 700, 2),
                                                              (24, 1024, 640, 13, 16), (1, 48, 10000, 2, 2400), (2, 72, 600, 257, 1)])
def test_cache_move_within_a_cache(layers, row_bytes, rows, count, most):
    rng = np.random.default_rng(rows)
    moves = disjoint_moves(rng, rows, count, most)
    keys, values = (torch.from_numpy(rng.integers(0, 256, (layers, rows, row_bytes), dtype=np.uint8)) for _ in range(2))
    device = keys.cuda(), values.cuda()
    cache = cache_of(*device)
    move(cache, cache, moves, layers, row_bytes)
    assert torch.equal(device[0].cpu(), moved(keys, keys, moves)) and torch.equal(device[1].cpu(), moved(values, values, moves))


@gpu
@pytest.mark.parametrize("offset,row_bytes", [(0, 64), (4, 64), (1, 33), (16, 2048)])
def test_cache_move_between_caches(offset, row_bytes):
    """A step's rows into pages, addresses and layer pitches that are no multiple of 16 bytes; other rows and the bytes
    between the layers stay. The same source row may be read twice."""
    rng, layers = np.random.default_rng(offset), 3
    flat = [torch.from_numpy(rng.integers(0, 256, 3 * 60 * row_bytes + 512, dtype=np.uint8)).cuda() for _ in range(4)]
    to = [t[offset:].as_strided((layers, 50, row_bytes), (55 * row_bytes + offset, row_bytes, 1)) for t in flat[:2]]
    source = [t[offset:].as_strided((layers, 9, row_bytes), (9 * row_bytes, row_bytes, 1)) for t in flat[2:]]
    before = [t.clone() for t in flat]
    moves = [(0, 49, 1), (1, 7, 1), (0, 8, 3), (5, 20, 4), (8, 0, 1), (3, 30, 0)]
    want = []
    for i in range(2):
        room = before[i].clone()
        view = room[offset:].as_strided((layers, 50, row_bytes), (55 * row_bytes + offset, row_bytes, 1))
        view.copy_(moved(view.clone(), source[i], moves))
        want.append(room)
    move(cache_of(*to), cache_of(*source), moves, layers, row_bytes)
    for i in range(2):
        assert torch.equal(flat[i], want[i]) and torch.equal(flat[i + 2], before[i + 2])


@gpu
def test_cache_move_in_a_graph_replays_its_moves():
    """The moves are read at the call: the host array may be gone or changed when a graph replays."""
    keys, values = (torch.arange(2 * 64 * 32, device="cuda").to(torch.uint8).view(2, 64, 32).clone() for _ in range(2))
    start = keys.clone()
    cache, moves = cache_of(keys, values), np.array([[0, 40, 3], [10, 50, 6]], dtype=np.int64)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        move(cache, cache, moves, 2, 32, torch.cuda.current_stream().cuda_stream)
    wanted = moved(start.cpu(), start.cpu(), moves.tolist())
    moves[:] = 0
    del moves
    for _ in range(3):
        keys.copy_(start)
        values.copy_(start)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(keys.cpu(), wanted) and torch.equal(values.cpu(), wanted)


@gpu
def test_cache_move_past_32_bits():
    """Rows whose bytes lie more than 2^32 from the cache's first."""
    row_bytes, rows = 1 << 16, 70000
    keys = torch.empty(1, rows, row_bytes, dtype=torch.uint8, device="cuda")
    values = torch.empty(1, rows, row_bytes, dtype=torch.uint8, device="cuda")
    assert rows * row_bytes > 1 << 32
    keys[0, 3], values[0, 3], keys[0, 69999], values[0, 69999] = 11, 22, 33, 44
    cache = cache_of(keys, values)
    move(cache, cache, [(3, 69000, 1), (69999, 4, 1)], 1, row_bytes)
    assert (keys[0, 69000] == 11).all() and (values[0, 69000] == 22).all() and (keys[0, 4] == 33).all() and (values[0, 4] == 44).all()


def host_cache(**changes):
    fields = dict(keys=1 << 20, values=1 << 24, rows=100, layer_pitch=6400)
    fields.update(changes)
    return native.CacheRows(**fields)


@pytest.mark.parametrize("to,source,layers,row_bytes,moves,message", [
    ({}, None, 0, 64, [], "layers"), ({}, None, 40000, 64, [], "layers"), ({}, None, 2, 0, [], "rows of at least"),
    (dict(keys=None), None, 2, 64, [], "null"), (dict(rows=0), None, 2, 64, [], "out of range"), (dict(rows=2**32), None, 2, 64, [], "out of range"),
    (dict(layer_pitch=6399), None, 2, 64, [], "layer pitch"), (dict(values=(1 << 20) + 64), None, 2, 64, [], "overlap"),
    ({}, dict(keys=(1 << 20) + 6400 * 2 - 1), 2, 64, [], "overlap"), ({}, dict(values=1 << 20, keys=1 << 28), 2, 64, [], "overlap"),
    ({}, None, 2, 64, [(-1, 5, 1)], "leaves"), ({}, None, 2, 64, [(0, 100, 1)], "leaves"), ({}, None, 2, 64, [(99, 5, 2)], "leaves"),
    ({}, None, 2, 64, [(0, 5, -1)], "leaves"), ({}, None, 2, 64, [(0, 5, 2**62)], "leaves"), ({}, None, 2, 64, [(2**62, 5, 1)], "leaves"),
    ({}, dict(keys=1 << 28, values=1 << 29, rows=3), 2, 64, [(2, 5, 2)], "leaves"),
    ({}, None, 2, 64, [(0, 5, 2), (10, 6, 1)], "twice"), ({}, None, 2, 64, [(0, 1, 2)], "twice"), ({}, None, 2, 64, [(0, 5, 1), (5, 9, 1)], "twice"),
    ({}, None, 2, 64, [(7, 7, 1)], "twice"), ({}, dict(keys=1 << 28, values=1 << 29), 2, 64, [(0, 5, 2), (10, 5, 2)], "twice"),
    ({}, None, 2, 64, [(60, 0, 30), (20, 40, 5), (41, 95, 1)], "twice"), ({}, dict(layer_pitch=9999), 1, 64, [(7, 7, 1)], "twice"),
    ({}, dict(layer_pitch=9999), 2, 64, [], "must be the same"), ({}, dict(rows=1 << 18, layer_pitch=1 << 24), 1, 64, [], "keys and values overlap"),
])
def test_cache_move_refusals(to, source, layers, row_bytes, moves, message):
    target = host_cache(**to)
    with pytest.raises(RuntimeError, match="cache_move: .*" + message):
        move(target, target if source is None else host_cache(**source), moves, layers, row_bytes)


def test_cache_move_of_nothing_launches_nothing():
    cache, error = host_cache(), ctypes.create_string_buffer(64)
    move(cache, cache, [], 2, 64)
    move(cache, cache, [(1, 2, 0), (1, 1, 0)], 2, 64)
    lib = native.library()
    assert lib.chroma_hip_cache_move(None, ctypes.byref(cache), 1, 64, None, 0, None, error, len(error)) == native.RUNTIME_ERROR
    assert lib.chroma_hip_cache_move(ctypes.byref(cache), ctypes.byref(cache), 1, 64, None, 1, None, error, len(error)) == native.RUNTIME_ERROR


# ------------------------------------------------------------------------------------------------ logit adjustments
def adjust_call(x, y, *, history=None, lengths=None, repetition=None, presence=None, frequency=None, bias=None, mask=None):
    rows, width = x.shape
    return native.Adjust(
        x=pointer(x), y=pointer(y), rows=rows, width=width, x_stride=x.stride()[0], y_stride=y.stride()[0], history=pointer(history),
        history_lengths=pointer(lengths), history_stride=0 if history is None else history.stride()[0],
        history_width=0 if history is None else history.shape[1], repetition=pointer(repetition), presence=pointer(presence),
        frequency=pointer(frequency), bias=pointer(bias), bias_stride=0 if bias is None or bias.dim() == 1 else bias.stride()[0],
        mask=pointer(mask), mask_stride=0 if mask is None or mask.dim() == 1 else mask.stride()[0], dtype=DTYPES[x.dtype])


def adjust(call, stream=None):
    error = ctypes.create_string_buffer(256)
    checked(native.library().chroma_hip_rows_adjust(ctypes.byref(call), stream, error, len(error)), error)


def adjust_reference(x, *, history=None, lengths=None, repetition=None, presence=None, frequency=None, bias=None, mask=None):
    """(result in 64 bits, bound of float arithmetic with one rounding per operation and one to x's type)."""
    rows, width = x.shape
    y = x.double().clone()
    off = torch.zeros_like(y)
    for r in range(rows):
        if history is not None:
            length = history.shape[1] if lengths is None else min(max(int(lengths[r]), 0), history.shape[1])
            ids = history[r, :length]
            ids, counts = torch.unique(ids[(ids >= 0) & (ids < width)], return_counts=True)
            rho, alpha, beta = (d if t is None else float(t[r]) for t, d in ((repetition, 1.0), (presence, 0.0), (frequency, 0.0)))
            old = y[r, ids]
            scaled = torch.where(old > 0, old / rho, old * rho)
            less = alpha + beta * counts.double()
            y[r, ids] = scaled - less
            # the quotient or product, beta * c, alpha + it, the difference
            off[r, ids] = 2.0**-24 * (scaled.abs() + abs(beta) * counts + (abs(alpha) + abs(beta) * counts) * 2 + (scaled - less).abs()) * 1.01
        if bias is not None:
            y[r] += (bias if bias.dim() == 1 else bias[r]).double()
            off[r] += 2.0**-24 * (y[r].abs() + off[r])
        if mask is not None:
            words = (mask if mask.dim() == 1 else mask[r]).numpy().view(np.uint32)
            blocked = torch.from_numpy(np.unpackbits(words.view(np.uint8), bitorder="little")[:width] == 0)
            y[r, blocked], off[r, blocked] = -math.inf, 0.0
    return y, off + torch.nan_to_num(y.abs(), posinf=0.0) * (HALF[x.dtype] if x.dtype == torch.bfloat16 else 0.0) * 1.01


def adjust_inputs(rows, width, history, dtype, seed, *, bias=None, mask=None):
    g = torch.Generator().manual_seed(seed)
    inputs = {"history": torch.randint(-2, width + 2, (rows, history), generator=g), "lengths": torch.randint(0, history + 1, (rows,), generator=g),
              "repetition": 0.5 + torch.rand(rows, generator=g), "presence": torch.randn(rows, generator=g), "frequency": torch.randn(rows, generator=g)}
    if history > 2:
        inputs["history"][:, ::2] = inputs["history"][:, :1]  # one id that makes up half of it
    shape = {None: None, "shared": (), "rows": (rows,)}
    if bias:
        inputs["bias"] = torch.randn(*shape[bias], width, generator=g)
    if mask:
        inputs["mask"] = torch.randint(-(2**31), 2**31, (*shape[mask], -(-width // 32)), generator=g).to(torch.int32)
    return (torch.randn(rows, width, generator=g) * 4).to(dtype), inputs


def check_adjust(x, inputs, in_place):
    want, bound = adjust_reference(x, **inputs)
    source = x.cuda()
    y = source if in_place else torch.full_like(source, 5.0)
    adjust(adjust_call(source, y, **on_gpu(inputs)))
    got = y.cpu().double()
    infinite = torch.isinf(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[infinite], want[infinite])
    fine = torch.isfinite(want)
    assert ((got - want).abs()[fine] <= bound[fine]).all()
    if not in_place:
        assert torch.equal(source.cpu().view(torch.uint8), x.view(torch.uint8))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("in_place", [False, True], ids=["apart", "in-place"])
@pytest.mark.parametrize("rows,width,history,bias,mask", [
    (1, 1, 1, None, None), (1, 33, 0, None, "shared"), (3, 100, 7, "shared", None), (2, 4097, 50, None, "rows"), (4, 1023, 300, "rows", "rows"),
    (1, 201088, 700, None, None), (2, 201088, 5000, "shared", "rows"), (5, 50001, 20000, "rows", "shared"), (70, 2049, 65, None, "rows"),
    (300, 515, 40, "shared", "shared"), (1, 700001, 9, None, None)])
def test_rows_adjust(rows, width, history, bias, mask, in_place, dtype):
    x, inputs = adjust_inputs(rows, width, history, dtype, rows + width, bias=bias, mask=mask)
    check_adjust(x, inputs, in_place)


@gpu
@pytest.mark.parametrize("in_place", [False, True], ids=["apart", "in-place"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_rows_adjust_special_values(dtype, in_place):
    """NaN and infinities stay or are masked, a row with every token blocked, a row with none, lengths outside the history,
    a repetition factor per sign, infinite biases; each parameter left out in turn."""
    x, inputs = adjust_inputs(6, 300, 20, dtype, 5, bias="shared", mask="rows")
    x[:, 10], x[:, 20], x[:, 30], x[:, 40], x[:, 41] = math.nan, math.inf, -math.inf, 0.0, torch.finfo(dtype).min
    inputs["history"][:, 0:5] = torch.tensor([10, 20, 30, 40, 41])
    inputs["mask"][0], inputs["mask"][1] = 0, -1
    inputs["bias"][50], inputs["bias"][51] = -math.inf, math.inf
    inputs["lengths"] = torch.tensor([-3, 2**40, 20, 0, 5, 19])
    check_adjust(x, inputs, in_place)
    for name in ("lengths", "repetition", "presence", "frequency", "bias", "mask"):
        check_adjust(x, {k: v for k, v in inputs.items() if k != name}, in_place)
    check_adjust(x, {"mask": inputs["mask"]}, in_place)
    check_adjust(x, {}, in_place)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("offset,x_stride,y_stride", [(0, 1000, 1000), (1, 1003, 1007), (3, 1001, 1032), (2, 1024, 1024)])
def test_rows_adjust_strides_and_neighbours(offset, x_stride, y_stride, dtype):
    """Rows that start off 16 bytes and end inside one; what lies beside them stays."""
    x, inputs = adjust_inputs(5, 999, 60, dtype, offset, bias="rows", mask="shared")
    want, bound = adjust_reference(x, **inputs)
    room = torch.full((offset + 5 * max(x_stride, y_stride) + 64,), 9.0, dtype=dtype, device="cuda")
    source, y = (torch.full_like(room, 9.0)[offset:].as_strided((5, 999), (s, 1)) for s in (x_stride, y_stride))
    source.copy_(x)
    device = on_gpu(inputs)
    device["bias"] = torch.full((5, 1010), math.nan, device="cuda")[:, 1:1000].copy_(device["bias"])
    device["history"] = torch.full((5, 64), 3, device="cuda", dtype=torch.int64)[:, 2:62].copy_(device["history"])
    adjust(adjust_call(source, y, **device))
    got = y.cpu().double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isinf(got), torch.isinf(want)) and ((got - want).abs()[fine] <= bound[fine]).all()
    storage = torch.as_strided(y, (len(room),), (1,), 0)
    written = torch.zeros(len(room), dtype=torch.bool, device="cuda")
    written[offset:].as_strided((5, 999), (y_stride, 1)).fill_(True)
    assert (storage[~written] == 9.0).all()


def plain_adjust_call(**changes):
    fields = dict(x=1 << 20, y=1 << 24, rows=2, width=100, x_stride=100, y_stride=100, history=1 << 25, history_lengths=None, history_stride=8,
                  history_width=8, repetition=None, presence=None, frequency=None, bias=1 << 26, bias_stride=0, mask=1 << 27, mask_stride=0,
                  dtype=native.FLOAT32)
    fields.update(changes)
    return native.Adjust(**fields)


@pytest.mark.parametrize("changes,message", [
    (dict(dtype=5), "dtype"), (dict(rows=0), "rows"), (dict(rows=65536), "rows"), (dict(width=0), "logits"), (dict(width=2**31), "logits"),
    (dict(x_stride=2**62), "out of range"), (dict(history_stride=2**41), "out of range"), (dict(x_stride=99), "stride"), (dict(y_stride=99), "stride"), (dict(history_stride=7), "stride"), (dict(history_width=-1), "stride"),
    (dict(bias_stride=50), "stride"), (dict(mask_stride=3), "stride"), (dict(x=None), "null"), (dict(y=None), "null"),
    (dict(x=(1 << 20) + 2), "own size"), (dict(y=(1 << 20) + 400), "apart"), (dict(y=1 << 20, y_stride=101), "apart"),
])
def test_rows_adjust_refusals(changes, message):
    with pytest.raises(RuntimeError, match="rows_adjust: .*" + message):
        adjust(plain_adjust_call(**changes))


def test_rows_adjust_refuses_no_call():
    error = ctypes.create_string_buffer(64)
    assert native.library().chroma_hip_rows_adjust(None, None, error, len(error)) == native.RUNTIME_ERROR


@gpu
def test_rows_adjust_in_a_graph():
    """A captured call reads the history, lengths and logits that lie there when it is replayed."""
    x, inputs = adjust_inputs(3, 5000, 40, torch.bfloat16, 8, bias="shared", mask="rows")
    device, source = on_gpu(inputs), x.cuda()
    y = torch.empty_like(source)
    adjust(adjust_call(source, y, **device))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        adjust(adjust_call(source, y, **device), torch.cuda.current_stream().cuda_stream)
    for turn in range(4):
        device["history"][:, turn] = 4999 - turn
        device["lengths"].fill_(10 * turn)
        y.fill_(0.0)
        graph.replay()
        torch.cuda.synchronize()
        eager = torch.empty_like(source)
        adjust(adjust_call(source, eager, **device))
        torch.cuda.synchronize()
        assert torch.equal(y.view(torch.int16), eager.view(torch.int16))
        inputs["history"], inputs["lengths"] = device["history"].cpu(), device["lengths"].cpu()
        want, bound = adjust_reference(x, **inputs)
        got, fine = y.cpu().double(), torch.isfinite(want)
        assert torch.equal(torch.isinf(got), torch.isinf(want)) and ((got - want).abs()[fine] <= bound[fine]).all()


# ------------------------------------------------------------------------------------------------ a run of them together
@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_decode_steps_of_the_operators(dtype):
    """Steps as a serving loop makes them, on a stream of its own: attention with the new rows, these rows stored into their
    pages (a branch's shared page copied first), logits from the result, adjusted by the tokens so far, the token chosen.
    Each attention against 64 bits over the text of its sequence, the stored rows bit for bit."""
    lib, g = native.library(), torch.Generator().manual_seed(6)
    kv, group, dim, page, pages, span, vocabulary = 2, 4, 32, 4, 40, 12, 2000
    lengths = [5, 8, 5]  # sequence 2 is a branch of sequence 0
    table = torch.full((3, span), -1, dtype=torch.int64)
    table[0, :2], table[1, :2], table[2, :2] = torch.tensor([7, 3]), torch.tensor([20, 11]), torch.tensor([7, 3])
    free = [page_id for page_id in range(pages) if page_id not in (7, 3, 20, 11)]
    k, v = (torch.randn(pages, page, kv, dim, generator=g).to(dtype) for _ in range(2))
    head = torch.randn(vocabulary, kv * group * dim, generator=g).to(dtype).cuda()
    k_device, v_device = k.cuda(), v.cuda()
    row_bytes = kv * dim * k.element_size()
    cache = native.CacheRows(keys=k_device.data_ptr(), values=v_device.data_ptr(), rows=pages * page, layer_pitch=pages * page * row_bytes)
    texts = [[1, 2, 3, 4, 5], [9] * 8, [1, 2, 3, 4, 5]]
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        for step in range(6):
            q = torch.randn(3, kv, group, dim, generator=g).to(dtype)
            k_new, v_new = (torch.randn(3, kv, dim, generator=g).to(dtype) for _ in range(2))
            inputs = {"q": q, "k_pages": k, "v_pages": v, "table": table, "lengths": torch.tensor(lengths), "k_new": k_new, "v_new": v_new}
            want, bound = attention_reference(**inputs, window=9, first=2)
            device = on_gpu({**inputs, "k_pages": None, "v_pages": None})
            out = torch.empty_like(device["q"])
            kept = attend(attention_call(**{**device, "k_pages": k_device, "v_pages": v_device}, out=out, window=9, first=2), stream.cuda_stream)
            moves = []
            for b in range(3):  # the pages of this step's rows
                i = lengths[b] // page
                if lengths[b] % page == 0:
                    table[b, i] = free.pop(0)
                elif b == 2 and step == 0:
                    moves.append((int(table[b, i]) * page, free[0] * page, lengths[b] % page))
                    k[free[0], : lengths[b] % page], v[free[0], : lengths[b] % page] = k[table[b, i], : lengths[b] % page], v[table[b, i], : lengths[b] % page]
                    table[b, i] = free.pop(0)
            move(cache, cache, moves, 1, row_bytes, stream.cuda_stream)
            fresh = native.CacheRows(keys=device["k_new"].data_ptr(), values=device["v_new"].data_ptr(), rows=3, layer_pitch=3 * row_bytes)
            move(cache, fresh, [(b, int(table[b, lengths[b] // page]) * page + lengths[b] % page, 1) for b in range(3)], 1, row_bytes, stream.cuda_stream)
            for b in range(3):
                k[table[b, lengths[b] // page], lengths[b] % page], v[table[b, lengths[b] // page], lengths[b] % page] = k_new[b], v_new[b]
            logits = out.reshape(3, -1) @ head.t().contiguous()
            longest = max(map(len, texts))
            history = torch.tensor([text + [-1] * (longest - len(text)) for text in texts])
            rules = {"history": history, "repetition": torch.full((3,), 1.3), "presence": torch.full((3,), 0.4),
                     "mask": torch.randint(-(2**31), 2**31, (3, -(-vocabulary // 32)), generator=g).to(torch.int32)}
            adjusted, on_device = torch.empty_like(logits), on_gpu(rules)
            adjust(adjust_call(logits, adjusted, **on_device), stream.cuda_stream)
            values, ids = torch.empty(3, 1, dtype=dtype, device="cuda"), torch.empty(3, 1, dtype=torch.int64, device="cuda")
            need, error = lib.chroma_hip_rows_topk_workspace(3, vocabulary, 1), ctypes.create_string_buffer(256)
            scratch = torch.empty(need, dtype=torch.uint8, device="cuda")
            checked(lib.chroma_hip_rows_topk(adjusted.data_ptr(), DTYPES[dtype], 3, vocabulary, 1, 1, values.data_ptr(), ids.data_ptr(),
                                             scratch.data_ptr(), need, stream.cuda_stream, error, len(error)), error)
            stream.synchronize()
            assert ((out.cpu().double() - want).abs() <= bound).all(), step
            assert torch.equal(k_device.cpu(), k) and torch.equal(v_device.cpu(), v)
            exact, off = adjust_reference(logits.cpu(), **rules)
            got, fine = adjusted.cpu().double(), torch.isfinite(exact)
            assert torch.equal(torch.isinf(got), torch.isinf(exact)) and ((got - exact).abs()[fine] <= off[fine]).all()
            for b in range(3):
                assert int(ids[b]) == int(torch.nonzero(got[b] == got[b].max())[0])
                texts[b].append(int(ids[b]))
                lengths[b] += 1
            del kept
