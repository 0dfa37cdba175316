"""The operators of batched decoding over a paged cache, at the sizes that serving meets.

* ``attention``: one new token per sequence over the pages of its cached keys and values
  (``chroma_hip_paged_attention``);
* ``move``: rows of a paged cache copied between caches or pages: a step's new rows stored, a sequence forked, the live
  pages compacted (``chroma_hip_cache_move``);
* ``adjust``: penalties for repeated tokens, biases and a grammar mask on logits (``chroma_hip_rows_adjust``).

Inputs lie on the GPU, as between two programs of a serving loop; what the host decides (page moves) is a host array.
"""

from __future__ import annotations

import ctypes
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
VOCABULARY = 201088


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one user of a GPT-OSS-20B-shaped model (8 KV heads of 8 query heads of 64): the smallest call, all latency
        {"name": "attention_1x900", "kind": "attention", "sequences": 1, "kv_heads": 8, "group": 8, "dim": 64, "longest": 900,
         "page": 16, "window": 0, "first": 0, "sinks": True, "fresh": True, "ragged": False, "dtype": "bf16"},
        # an ordinary batch of conversations of mixed lengths on the same layer
        {"name": "attention_32x4096", "kind": "attention", "sequences": 32, "kv_heads": 8, "group": 8, "dim": 64, "longest": 4096,
         "page": 16, "window": 0, "first": 0, "sinks": True, "fresh": True, "ragged": True, "dtype": "bf16"},
        # its sliding-window layers, the first tokens kept visible
        {"name": "attention_64x8192_window", "kind": "attention", "sequences": 64, "kv_heads": 8, "group": 8, "dim": 64,
         "longest": 8192, "page": 32, "window": 128, "first": 4, "sinks": True, "fresh": True, "ragged": True, "dtype": "bf16"},
        # a few very long documents, heads of 128, large pages, no new row (it was stored first)
        {"name": "attention_6x131072", "kind": "attention", "sequences": 6, "kv_heads": 8, "group": 4, "dim": 128, "longest": 131072,
         "page": 64, "window": 0, "first": 0, "sinks": False, "fresh": False, "ragged": True, "dtype": "bf16"},
        # the dev model's heads (one KV head of 8 heads of 16) in float32, a page length that is no power of two
        {"name": "attention_20x513_f32", "kind": "attention", "sequences": 20, "kv_heads": 1, "group": 8, "dim": 16, "longest": 513,
         "page": 12, "window": 0, "first": 0, "sinks": True, "fresh": True, "ragged": True, "dtype": "f32"},
        # a decode step's new rows of 64 sequences stored into their pages, 24 layers
        {"name": "move_step_64", "kind": "move", "use": "step", "layers": 24, "row_bytes": 1024, "page": 16, "pages": 4096, "moves": 64},
        # 24 branches of a prompt: each gets a copy of the prompt's last, partly filled page
        {"name": "move_fork_24", "kind": "move", "use": "fork", "layers": 24, "row_bytes": 1024, "page": 16, "pages": 4096, "moves": 24},
        # the live pages of a fragmented cache brought to its front
        {"name": "move_compact_1500", "kind": "move", "use": "compact", "layers": 24, "row_bytes": 1024, "page": 16, "pages": 6000,
         "moves": 1500},
        # one conversation's row: penalties over its history, nothing masked
        {"name": "adjust_1_f32", "kind": "adjust", "rows": 1, "width": VOCABULARY, "history": 700, "bias": False, "mask": False,
         "dtype": "f32"},
        # a batch under grammars (a mask each) with a shared bias
        {"name": "adjust_64_bf16", "kind": "adjust", "rows": 64, "width": VOCABULARY, "history": 4096, "bias": True, "mask": True, "dtype": "bf16"},
        # the largest batch, float logits, a vocabulary of odd width
        {"name": "adjust_256_f32", "kind": "adjust", "rows": 256, "width": 100003, "history": 2000, "bias": True, "mask": True, "dtype": "f32"},
    ]


def _log_uniform(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "move", "adjust", "adjust"])
    if kind == "attention":
        kv_heads, group, dim = rng.choice([(8, 8, 64), (8, 8, 64), (8, 4, 128), (4, 7, 128), (1, 8, 16), (2, 3, 80), (16, 1, 64), (2, 16, 32)])
        dtype = rng.choice(["bf16", "bf16", "f32"])
        sequences = _log_uniform(rng, 1, 128)
        # no more cached bytes than the largest listed case reads
        most = 6 * 131072 * 8 * 128 * 2 // (sequences * kv_heads * dim * (2 if dtype == "bf16" else 4))
        return {"kind": kind, "sequences": sequences, "kv_heads": kv_heads, "group": group, "dim": dim,
                "longest": _log_uniform(rng, 1, min(65536, most)), "page": rng.choice([1, 7, 12, 16, 16, 32, 64, 128]),
                "window": rng.choice([0, 0, 0, 128, 1000]), "first": rng.choice([0, 0, 4, 33]), "sinks": rng.random() < 0.5,
                "fresh": rng.random() < 0.7, "ragged": rng.random() < 0.8, "dtype": dtype}
    if kind == "move":
        use = rng.choice(["step", "fork", "compact"])
        page, pages, layers = rng.choice([1, 8, 12, 16, 32]), _log_uniform(rng, 512, 2048), rng.randint(1, 24)
        row_bytes = rng.choice([64, 256, 1000, 1024, 2048])
        most = min(pages // 3, 1500 * 16 * 24 * 1024 // (page * layers * row_bytes))  # no more bytes than the largest listed case
        return {"kind": kind, "use": use, "layers": layers, "row_bytes": row_bytes, "page": page, "pages": pages,
                "moves": _log_uniform(rng, 1, most if use == "compact" else 128)}
    width = _log_uniform(rng, 50, VOCABULARY)
    return {"kind": kind, "rows": _log_uniform(rng, 1, min(256, 256 * 100003 // width)), "width": width, "history": _log_uniform(rng, 1, 8192),
            "bias": rng.random() < 0.5, "mask": rng.random() < 0.5, "dtype": rng.choice(["f32", "bf16"])}


# ------------------------------------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _lengths(case, g):
    """Cached rows of each sequence: all of the longest, or a mix of short and long ones with one of the longest."""
    n, longest = case["sequences"], case["longest"]
    if not case["ragged"]:
        return torch.full((n,), longest, dtype=torch.int64, device="cuda")
    share = torch.rand(n, generator=g, device="cuda")
    lengths = (share * longest).long()
    lengths[0] = longest
    return lengths


def _prepare_attention(case, g):
    n, kv, group, dim, page = case["sequences"], case["kv_heads"], case["group"], case["dim"], case["page"]
    dtype = DTYPES[case["dtype"]]
    span = -(-case["longest"] // page)
    lengths = _lengths(case, g)
    used = (lengths + page - 1) // page
    slots = torch.arange(span, device="cuda")[None, :] < used[:, None]
    pages = n * span + 3
    table = torch.full((n, span), -1, dtype=torch.int64, device="cuda")
    table[slots] = torch.randperm(pages, generator=g, device="cuda")[: int(slots.sum())]

    def values(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)

    state = {"q": values(n, kv, group, dim), "k_pages": torch.empty(pages, page, kv, dim, dtype=dtype, device="cuda"),
             "v_pages": torch.empty(pages, page, kv, dim, dtype=dtype, device="cuda"), "table": table, "lengths": lengths,
             "k_new": values(n, kv, dim) if case["fresh"] else None, "v_new": values(n, kv, dim) if case["fresh"] else None,
             "sinks": values(kv * group) if case["sinks"] else None, "scale": dim**-0.5}
    for cache in (state["k_pages"], state["v_pages"]):
        cache.normal_(generator=g)
    return state


def _page_moves(case, rng):
    """Host array [moves, 3]: first source row, first destination row, rows."""
    page, pages, count = case["page"], case["pages"], case["moves"]
    if case["use"] == "step":  # row i of the step goes to some place of a page of its own
        targets = rng.choice(pages, count, replace=False)
        return np.stack([np.arange(count), targets * page + rng.integers(0, page, count), np.ones(count)], 1).astype(np.int64)
    if case["use"] == "fork":  # the filled rows of the parents' last pages, to new pages
        chosen = rng.choice(pages, count + 1 + count // 16, replace=False)
        parents = chosen[count:][rng.integers(0, len(chosen) - count, count)]
        filled = rng.integers(1, page + 1, pages)[parents]
        return np.stack([parents * page, chosen[:count] * page, filled], 1).astype(np.int64)
    live = np.sort(rng.choice(np.arange(pages // 3, pages), count, replace=False))  # the front third has room for them
    holes = np.sort(rng.choice(pages // 3, count, replace=False))
    return np.stack([live * page, holes * page, np.full(count, page)], 1).astype(np.int64)


def _prepare_move(case, seed, g):
    moves = _page_moves(case, np.random.default_rng(seed))

    def cache(rows):
        return torch.randint(0, 256, (case["layers"], rows, case["row_bytes"]), generator=g, device="cuda", dtype=torch.uint8)

    rows = case["pages"] * case["page"]
    state = {"keys": cache(rows), "values": cache(rows), "moves": moves}
    state["new_keys"], state["new_values"] = (cache(case["moves"]), cache(case["moves"])) if case["use"] == "step" else (None, None)
    return state


def _prepare_adjust(case, g):
    rows, width, history = case["rows"], case["width"], case["history"]
    logits = (torch.randn(rows, width, generator=g, device="cuda") * 3).to(DTYPES[case["dtype"]])
    # a text's tokens: few ids make up most of it
    ids = (torch.rand(rows, history, generator=g, device="cuda").pow(6) * width).long().clamp_(max=width - 1)
    lengths = (torch.rand(rows, generator=g, device="cuda") * (history + 1)).long().clamp_(max=history)
    lengths[0] = history
    ids[torch.arange(history, device="cuda")[None, :] >= lengths[:, None]] = -1
    state = {"logits": logits, "history": ids, "lengths": lengths,
             "repetition": 1 + torch.rand(rows, generator=g, device="cuda") * 0.3,
             "presence": torch.rand(rows, generator=g, device="cuda"), "frequency": torch.rand(rows, generator=g, device="cuda") * 0.2,
             "bias": None, "mask": None}
    if case["bias"]:
        bias = torch.zeros(width, device="cuda")
        some = torch.randperm(width, generator=g, device="cuda")[:300]
        bias[some] = torch.randn(len(some), generator=g, device="cuda") * 5
        state["bias"] = bias
    if case["mask"]:
        words = -(-width // 32)
        state["mask"] = torch.randint(-(2**31), 2**31, (rows, words), generator=g, device="cuda", dtype=torch.int64).to(torch.int32)
    return state


def prepare(case, seed):
    g = _generator(seed)
    if case["kind"] == "move":
        state = _prepare_move(case, seed, g)
    else:
        state = (_prepare_attention if case["kind"] == "attention" else _prepare_adjust)(case, g)
    state["case"] = case
    return state


# ------------------------------------------------------------------------------------------------ the plain forms
def _visible(case, lengths, keys):
    """[sequences, keys]: whether cached row j is seen by the new token."""
    j = torch.arange(keys, device=lengths.device)[None, :]
    seen = j < lengths[:, None]
    if case["window"]:
        last = lengths[:, None] - (0 if case["fresh"] else 1)
        seen = seen & ((j > last - case["window"]) | (j < case["first"]))
    return seen


def _attention_plain(state):
    case, table = state["case"], state["table"]
    n, kv, group, dim = state["q"].shape
    keys = table.shape[1] * case["page"]
    where = table.clamp(min=0)
    # [sequences, KV, D, keys] and [sequences, KV, keys, D]
    k = state["k_pages"][where].float().reshape(n, keys, kv, dim).permute(0, 2, 3, 1).contiguous()
    v = state["v_pages"][where].float().reshape(n, keys, kv, dim).transpose(1, 2).contiguous()
    q = state["q"].float() * state["scale"]
    seen = _visible(case, state["lengths"], keys)[:, None, None, :]
    scores = torch.matmul(q, k).masked_fill(~seen, -math.inf)
    fresh = torch.full_like(scores[..., :1], -math.inf)
    if state["k_new"] is not None:
        fresh = (q * state["k_new"].float()[:, :, None, :]).sum(-1, keepdim=True)
    sink = torch.full_like(fresh, -math.inf) if state["sinks"] is None else state["sinks"].float().reshape(1, kv, group, 1).expand_as(fresh)
    top = torch.maximum(torch.maximum(scores.amax(-1, keepdim=True), fresh), sink)
    top = torch.where(top == -math.inf, 0.0, top)
    weights = torch.exp(scores - top)
    total = weights.sum(-1, keepdim=True) + torch.exp(fresh - top) + torch.exp(sink - top)
    mixed = torch.matmul(weights, v)
    if state["v_new"] is not None:
        mixed = mixed + torch.exp(fresh - top) * state["v_new"].float()[:, :, None, :]
    return torch.where(total > 0, mixed / total, 0.0).to(state["q"].dtype)


def _move_plain(state):
    moves = torch.from_numpy(state["moves"]).cuda()
    most = int(state["moves"][:, 2].max())
    step = torch.arange(most, device="cuda")[None, :]
    taken = step < moves[:, 2:3]
    source, target = (moves[:, 0:1] + step)[taken], (moves[:, 1:2] + step)[taken]
    for cache, new in ((state["keys"], state["new_keys"]), (state["values"], state["new_values"])):
        cache[:, target] = (cache if new is None else new)[:, source]
    return [state["keys"], state["values"]]


def _adjust_plain(state):
    x = state["logits"].float()
    rows, width = x.shape
    ids = state["history"]
    counted = (torch.arange(ids.shape[1], device="cuda")[None, :] < state["lengths"][:, None]) & (ids >= 0) & (ids < width)
    counts = torch.zeros(rows, width, dtype=torch.int32, device="cuda")
    counts.scatter_add_(1, torch.where(counted, ids, 0), counted.to(torch.int32))
    seen = counts > 0
    repetition = state["repetition"][:, None]
    y = torch.where(seen, torch.where(x > 0, x / repetition, x * repetition), x)
    y = y - torch.where(seen, state["presence"][:, None] + state["frequency"][:, None] * counts, 0.0)
    if state["bias"] is not None:
        y = y + state["bias"]
    if state["mask"] is not None:
        bits = (state["mask"][:, :, None] >> torch.arange(32, dtype=torch.int32, device="cuda")) & 1
        y = y.masked_fill(bits.reshape(rows, -1)[:, :width] == 0, -math.inf)
    return y.to(state["logits"].dtype)


# ------------------------------------------------------------------------------------------------ the framework's calls
def _pointer(tensor):
    return None if tensor is None else tensor.data_ptr()


def _checked(status, error):
    from chroma_amd._src import native

    native.check(status, error)


def _attention_own(state):
    from chroma_amd._src import native

    lib, case, error = native.library(), state["case"], ctypes.create_string_buffer(256)
    n, kv, group, dim = state["q"].shape
    out = torch.empty_like(state["q"])
    call = native.PagedAttention(
        q=state["q"].data_ptr(), k_pages=state["k_pages"].data_ptr(), v_pages=state["v_pages"].data_ptr(), k_new=_pointer(state["k_new"]),
        v_new=_pointer(state["v_new"]), sinks=_pointer(state["sinks"]), table=state["table"].data_ptr(), lengths=state["lengths"].data_ptr(),
        out=out.data_ptr(), sequences=n, kv_heads=kv, group=group, dim=dim, pages=state["k_pages"].shape[0], page_rows=case["page"],
        page_stride=case["page"] * kv * dim, row_stride=kv * dim, head_stride=dim, q_stride=kv * group * dim, new_stride=kv * dim,
        out_stride=kv * group * dim, table_stride=state["table"].shape[1], longest=case["longest"], window=case["window"],
        first=case["first"], scale=state["scale"], dtype=native.FLOAT32 if out.dtype == torch.float32 else native.BFLOAT16)
    if "workspace" not in state:  # a serving loop keeps it
        need = lib.chroma_hip_paged_attention_workspace(ctypes.byref(call))
        state["workspace"] = torch.empty(max(1, need), dtype=torch.uint8, device="cuda")
    _checked(lib.chroma_hip_paged_attention(ctypes.byref(call), state["workspace"].data_ptr(), state["workspace"].numel(),
                                            torch.cuda.current_stream().cuda_stream, error, len(error)), error)
    return out


def _move_own(state):
    from chroma_amd._src import native

    lib, error, moves = native.library(), ctypes.create_string_buffer(256), state["moves"]

    def rows_of(keys, values):
        return native.CacheRows(keys=keys.data_ptr(), values=values.data_ptr(), rows=keys.shape[1], layer_pitch=keys.shape[1] * keys.shape[2])

    cache = rows_of(state["keys"], state["values"])
    source = cache if state["new_keys"] is None else rows_of(state["new_keys"], state["new_values"])
    layers, _, row_bytes = state["keys"].shape
    _checked(lib.chroma_hip_cache_move(ctypes.byref(cache), ctypes.byref(source), layers, row_bytes, moves.ctypes.data, len(moves),
                                       torch.cuda.current_stream().cuda_stream, error, len(error)), error)
    return [state["keys"], state["values"]]


def _adjust_own(state):
    from chroma_amd._src import native

    lib, error, x = native.library(), ctypes.create_string_buffer(256), state["logits"]
    rows, width = x.shape
    y, mask = torch.empty_like(x), state["mask"]
    call = native.Adjust(
        x=x.data_ptr(), y=y.data_ptr(), rows=rows, width=width, x_stride=width, y_stride=width, history=state["history"].data_ptr(),
        history_lengths=state["lengths"].data_ptr(), history_stride=state["history"].shape[1], history_width=state["history"].shape[1],
        repetition=state["repetition"].data_ptr(), presence=state["presence"].data_ptr(), frequency=state["frequency"].data_ptr(),
        bias=_pointer(state["bias"]), bias_stride=0, mask=_pointer(mask), mask_stride=0 if mask is None else mask.shape[1],
        dtype=native.FLOAT32 if x.dtype == torch.float32 else native.BFLOAT16)
    _checked(lib.chroma_hip_rows_adjust(ctypes.byref(call), torch.cuda.current_stream().cuda_stream, error, len(error)), error)
    return y


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"attention": _attention_own, "move": _move_own, "adjust": _adjust_own}[kind](state)
    if kind == "attention":
        return _attention_plain(state)
    if kind == "move":
        return _move_plain(state)
    return _adjust_plain(state)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["kind"] == "attention":
        size = 4 if case["dtype"] == "f32" else 2
        # the mean of the lengths that prepare() draws, cut by the window
        keys = case["longest"] * (0.5 if case["ragged"] else 1.0)
        if case["window"]:
            keys = min(keys, case["window"] + case["first"])
        heads = case["sequences"] * case["kv_heads"]
        rows = heads * case["group"] * case["dim"]
        fresh = 2 * heads * case["dim"] * size if case["fresh"] else 0
        return {"bytes": 2 * heads * keys * case["dim"] * size + 2 * rows * size + fresh + case["sequences"] * 8 * (keys / case["page"] + 1),
                "flops": 4 * rows * keys}
    if case["kind"] == "move":
        rows = case["moves"] * (1 if case["use"] == "step" else (case["page"] + 1) / 2 if case["use"] == "fork" else case["page"])
        return {"bytes": 4 * case["layers"] * rows * case["row_bytes"], "flops": 0}
    size = 4 if case["dtype"] == "f32" else 2
    elements = case["rows"] * case["width"]
    read = elements * size + case["rows"] * case["history"] * 4 + (case["width"] * 4 if case["bias"] else 0) + (elements / 8 if case["mask"] else 0)
    return {"bytes": read + elements * size, "flops": 4 * elements}


# ------------------------------------------------------------------------------------------------ 64 bits, by the definitions
def _attention_exact(state):
    """Sequence by sequence: the visible rows in order, a softmax over them, the sum of their values."""
    case, page = state["case"], state["case"]["page"]
    n, kv, group, dim = state["q"].shape
    result = torch.zeros(n, kv, group, dim, dtype=torch.float64, device="cuda")
    for b, length in enumerate(state["lengths"].tolist()):
        j = torch.arange(length, device="cuda")
        if case["window"]:
            now = length if case["fresh"] else length - 1
            j = j[(now - j < case["window"]) | (j < case["first"])]
        place = state["table"][b][j // page] * page + j % page
        for h in range(kv):
            k = state["k_pages"].view(-1, kv, dim)[place, h].double()
            v = state["v_pages"].view(-1, kv, dim)[place, h].double()
            if state["k_new"] is not None:
                k, v = torch.cat([k, state["k_new"][b, h].double()[None]]), torch.cat([v, state["v_new"][b, h].double()[None]])
            if not len(k):
                continue
            s = torch.mm(state["q"][b, h].double(), k.t().contiguous()) * state["scale"]
            if state["sinks"] is not None:
                s = torch.cat([s, state["sinks"].double().view(kv, group)[h][:, None]], 1)
            p = torch.softmax(s, 1)[:, : len(k)]
            result[b, h] = torch.mm(p, v)
    return result


def _adjust_exact(state):
    """Row by row, each distinct token of the history in turn."""
    x = state["logits"].double().cpu().numpy()
    rows, width = x.shape
    y = x.copy()
    history, lengths = state["history"].cpu().numpy(), state["lengths"].cpu().numpy()
    repetition, presence, frequency = (state[name].double().cpu().numpy() for name in ("repetition", "presence", "frequency"))
    for r in range(rows):
        ids, times = np.unique(history[r, : lengths[r]], return_counts=True)
        times, ids = times[(ids >= 0) & (ids < width)], ids[(ids >= 0) & (ids < width)]
        old = x[r, ids]
        y[r, ids] = np.where(old > 0, old / repetition[r], old * repetition[r]) - presence[r] - frequency[r] * times
    if state["bias"] is not None:
        y += state["bias"].double().cpu().numpy()
    if state["mask"] is not None:
        words = state["mask"].cpu().numpy().view(np.uint32)
        allowed = np.unpackbits(words.view(np.uint8), axis=1, bitorder="little")[:, :width]
        y[allowed == 0] = -np.inf
    return torch.from_numpy(y)


def exact(case, seed):
    if case["kind"] == "move":
        return None  # whole values: equal or not
    state = prepare(case, seed)
    return _attention_exact(state) if case["kind"] == "attention" else _adjust_exact(state)
