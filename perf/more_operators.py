"""The operators of a serving step whose sequences take any number of tokens, at the sizes that serving meets.

* ``plan``: page tables, slots, positions and row starts made from the requests' lengths (``chroma_hip_paged_plan``);
* ``store``: new rows of keys and values stored at their slots (``chroma_hip_cache_store``);
* ``chunk``: attention of a chunk of new tokens of every sequence over a paged cache (``chroma_hip_paged_chunk_attention``);
* ``sample``: a token drawn from each row of logits under temperature, top-k, top-p and min-p (``chroma_hip_rows_sample``).

Everything lies on the GPU, as inside a serving step that asks the host nothing.
"""

from __future__ import annotations

import ctypes
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
VOCABULARY = 201088


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one user's short second turn on a GPT-OSS-20B-shaped layer (8 KV heads of 8 heads of 64): all latency
        {"name": "chunk_1x16_after_900", "kind": "chunk", "sequences": 1, "kv_heads": 8, "group": 8, "dim": 64, "chunk": 16, "longest": 900,
         "page": 16, "window": 0, "first": 0, "sinks": True, "fresh": True, "mix": "even", "dtype": "bf16"},
        # an ordinary step on the same layer: a quarter of the sequences bring prompt chunks, the others decode one token
        {"name": "chunk_32x512_mixed", "kind": "chunk", "sequences": 32, "kv_heads": 8, "group": 8, "dim": 64, "chunk": 512, "longest": 4096,
         "page": 16, "window": 0, "first": 0, "sinks": True, "fresh": True, "mix": "serving", "dtype": "bf16"},
        # its sliding-window layers, rows stored first, the first tokens kept visible
        {"name": "chunk_8x1000_window", "kind": "chunk", "sequences": 8, "kv_heads": 8, "group": 8, "dim": 64, "chunk": 1000, "longest": 5000,
         "page": 32, "window": 128, "first": 4, "sinks": True, "fresh": False, "mix": "ragged", "dtype": "bf16"},
        # the largest: long documents taken in chunks of 2048, heads of 128
        {"name": "chunk_2x2048_after_30000", "kind": "chunk", "sequences": 2, "kv_heads": 8, "group": 4, "dim": 128, "chunk": 2048,
         "longest": 30000, "page": 64, "window": 0, "first": 0, "sinks": False, "fresh": True, "mix": "even", "dtype": "bf16"},
        # the dev model's heads (one KV head of 8 heads of 16) in float32, a page length that is no power of two
        {"name": "chunk_20x61_f32", "kind": "chunk", "sequences": 20, "kv_heads": 1, "group": 8, "dim": 16, "chunk": 61, "longest": 513,
         "page": 12, "window": 0, "first": 0, "sinks": True, "fresh": True, "mix": "ragged", "dtype": "f32"},
        # a decode step's plan: a token of each of 64 sequences
        {"name": "plan_64x1", "kind": "plan", "sequences": 64, "chunk": 1, "longest": 4096, "page": 16, "span": 272},
        # a large batch of prompts and continued texts
        {"name": "plan_1024x80", "kind": "plan", "sequences": 1024, "chunk": 80, "longest": 16000, "page": 16, "span": 1024},
        # one layer's new rows of a decode step, out of the fused projection's rows
        {"name": "store_64x1", "kind": "store", "tokens": 64, "layers": 1, "row_bytes": 1024, "pitch": 10240, "rows": 65536},
        # a prompt step's rows in all 24 layers
        {"name": "store_8000x24", "kind": "store", "tokens": 8000, "layers": 24, "row_bytes": 1024, "pitch": 1024, "rows": 16384},
        # one conversation, every filter on
        {"name": "sample_1_f32", "kind": "sample", "rows": 1, "width": VOCABULARY, "filters": "all", "dtype": "f32"},
        # a batch whose users chose their own settings, some of them the largest logit
        {"name": "sample_64_bf16", "kind": "sample", "rows": 64, "width": VOCABULARY, "filters": "mixed", "dtype": "bf16"},
        # the largest batch, whole distributions (temperature alone), a vocabulary of odd width
        {"name": "sample_256_f32", "kind": "sample", "rows": 256, "width": 100003, "filters": "none", "dtype": "f32"},
    ]


def _log_uniform(rng, low, high):
    high = max(low, high)
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    kind = rng.choice(["chunk", "chunk", "chunk", "sample", "sample", "plan", "store"])
    if kind == "chunk":
        kv_heads, group, dim = rng.choice([(8, 8, 64), (8, 8, 64), (8, 4, 128), (4, 7, 128), (1, 8, 16), (2, 3, 80), (16, 1, 64), (2, 16, 32), (4, 2, 256)])
        dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
        sequences, mix = _log_uniform(rng, 1, 64), rng.choice(["even", "ragged", "serving"])
        # no more (token, key) pairs of heads than the largest listed case; float32 products are slower by more than eight times
        most = (2 * 2048 * 32 * 31000) // (sequences * kv_heads * group * max(1, dim // 128)) // (1 if dtype == "bf16" else 8)
        chunk = _log_uniform(rng, 1, min(2048, int(math.sqrt(most))))
        return {"kind": kind, "sequences": sequences, "kv_heads": kv_heads, "group": group, "dim": dim, "chunk": chunk,
                "longest": _log_uniform(rng, chunk, min(30000, most // chunk - chunk)), "page": rng.choice([1, 7, 12, 16, 16, 32, 64, 128]),
                "window": rng.choice([0, 0, 0, 128, 1000]), "first": rng.choice([0, 0, 4, 33]), "sinks": rng.random() < 0.5,
                "fresh": rng.random() < 0.6, "mix": mix, "dtype": dtype}
    if kind == "plan":
        page, longest, chunk = rng.choice([1, 8, 12, 16, 16, 64]), _log_uniform(rng, 1, 16000), _log_uniform(rng, 1, 512)
        span = -(-(longest + chunk) // page) + rng.randint(0, 9)
        return {"kind": kind, "sequences": _log_uniform(rng, 1, min(1024, 1024 * 80 // chunk, (1 << 22) // span)), "chunk": chunk,
                "longest": longest, "page": page, "span": span}
    if kind == "store":
        row_bytes, layers = rng.choice([64, 256, 1000, 1024, 2048]), rng.randint(1, 24)
        tokens = _log_uniform(rng, 1, min(8000, 8000 * 24 * 1024 // (layers * row_bytes)))
        return {"kind": kind, "tokens": tokens, "layers": layers, "row_bytes": row_bytes,
                "pitch": row_bytes + rng.choice([0, 0, 16, 1024, 5000]), "rows": tokens + _log_uniform(rng, 1, 8000)}
    width = _log_uniform(rng, 50, VOCABULARY)
    return {"kind": kind, "rows": _log_uniform(rng, 1, min(256, 256 * 100003 // width)), "width": width,
            "filters": rng.choice(["all", "mixed", "mixed", "none"]), "dtype": rng.choice(["f32", "bf16"])}


# ------------------------------------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _counts(case):
    """New tokens of each sequence: all the same, of any length, or a quarter prompts and the others one token. The case alone
    says them, as a step's shape is known where its program is called."""
    n, chunk = case["sequences"], case["chunk"]
    if case["mix"] == "even":
        return [chunk] * n
    rng = random.Random(n * 1000003 + chunk)
    return [chunk if b == 0 else 1 if case["mix"] == "serving" and b >= (n + 3) // 4 else rng.randint(0, chunk) for b in range(n)]


def _prepare_chunk(case, g):
    n, kv, group, dim, page = case["sequences"], case["kv_heads"], case["group"], case["dim"], case["page"]
    dtype = DTYPES[case["dtype"]]
    counts = torch.tensor(_counts(case), dtype=torch.int64, device="cuda")
    lengths = torch.full((n,), case["longest"], dtype=torch.int64, device="cuda")
    if case["mix"] != "even":
        lengths = (torch.rand(n, generator=g, device="cuda") * (case["longest"] + 1)).long().clamp_(max=case["longest"])
        lengths[0] = case["longest"]
    if not case["fresh"]:  # the new rows are among them
        lengths = torch.maximum(lengths, counts)
    span = -(-case["longest"] // page)
    slots = torch.arange(span, device="cuda")[None, :] < ((lengths + page - 1) // page)[:, None]
    pages = n * span + 3
    table = torch.full((n, span), -1, dtype=torch.int64, device="cuda")
    table[slots] = torch.randperm(pages, generator=g, device="cuda")[: int(slots.sum())]
    starts = torch.zeros(n + 1, dtype=torch.int64, device="cuda")
    starts[1:] = counts.cumsum(0)
    tokens = int(starts[-1])

    def values(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)

    state = {"q": values(tokens, kv, group, dim), "k_pages": torch.empty(pages, page, kv, dim, dtype=dtype, device="cuda"),
             "v_pages": torch.empty(pages, page, kv, dim, dtype=dtype, device="cuda"), "table": table, "lengths": lengths, "starts": starts,
             "k_new": values(tokens, kv, dim) if case["fresh"] else None, "v_new": values(tokens, kv, dim) if case["fresh"] else None,
             "sinks": values(kv * group) if case["sinks"] else None, "scale": dim**-0.5}
    for cache in (state["k_pages"], state["v_pages"]):
        cache.normal_(generator=g)
    return state


def _prepare_plan(case, g):
    n, page, span = case["sequences"], case["page"], case["span"]
    counts = torch.ones(n, dtype=torch.int64, device="cuda")
    if case["chunk"] > 1:  # some requests wait
        counts = (torch.rand(n, generator=g, device="cuda") * (case["chunk"] + 1)).long().clamp_(max=case["chunk"])
    lengths = (torch.rand(n, generator=g, device="cuda") * (case["longest"] + 1)).long().clamp_(max=case["longest"])
    held = (lengths + page - 1) // page
    wanted = (lengths + counts + page - 1) // page - held
    pages = n * span + 1 + n // 8
    order = torch.randperm(pages, generator=g, device="cuda")
    slots = torch.arange(span, device="cuda")[None, :] < held[:, None]
    table = torch.full((n, span), -1, dtype=torch.int64, device="cuda")
    used = int(held.sum())
    table[slots] = order[:used]
    spare = int(wanted.sum()) + 1 + n // 8
    return {"lengths": lengths, "counts": counts, "table": table, "free": order[used: used + 7 + spare].contiguous(),
            "cursor": torch.tensor([min(5, max(0, len(order) - used - spare))], dtype=torch.int64, device="cuda"), "pages": pages,
            "tokens": n * case["chunk"]}


def _prepare_store(case, g):
    tokens, layers, row, pitch, rows = (case[name] for name in ("tokens", "layers", "row_bytes", "pitch", "rows"))

    def noise(*shape):
        return torch.randint(0, 256, shape, generator=g, device="cuda", dtype=torch.uint8)

    slots = torch.randperm(rows, generator=g, device="cuda")[:tokens].contiguous()
    slots[torch.rand(tokens, generator=g, device="cuda") < 0.05] = -1  # a padded batch's rows that belong to no sequence
    return {"keys": noise(layers, rows, row), "values": noise(layers, rows, row), "new_keys": noise(layers, tokens, pitch)[:, :, :row],
            "new_values": noise(layers, tokens, pitch)[:, :, :row], "slots": slots}


def _prepare_sample(case, g):
    rows, width = case["rows"], case["width"]

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    # a text's next token: a wide bulk, and some tokens of increasing likelihood above it
    logits = torch.randn(rows, width, generator=g, device="cuda") * 2
    few = min(width, 200)
    logits[:, torch.randperm(width, generator=g, device="cuda")[:few]] += -2.5 * torch.log(uniform(rows, few).clamp_(min=1e-6))
    logits[uniform(rows, width) < 0.01] = -math.inf  # tokens that a grammar leaves out
    state = {"logits": logits.to(DTYPES[case["dtype"]]), "uniform": uniform(rows), "temperature": 0.3 + 1.2 * uniform(rows),
             "top_k": None, "top_p": None, "min_p": None}
    if case["filters"] != "none":
        choice = torch.tensor([0, 1, 20, 40, 50, 200, 1000], device="cuda")
        state["top_k"] = choice[torch.randint(0, len(choice), (rows,), generator=g, device="cuda")]
        state["top_p"] = torch.where(uniform(rows) < 0.3, 1.0, 0.5 + 0.49 * uniform(rows))
        state["min_p"] = torch.where(uniform(rows) < 0.5, 0.0, 0.1 * uniform(rows))
        if case["filters"] == "all":
            state["top_k"].fill_(50)
            state["top_p"].fill_(0.9)
            state["min_p"].fill_(0.02)
        else:
            state["temperature"][uniform(rows) < 0.1] = 0.0
    return state


def prepare(case, seed):
    make = {"chunk": _prepare_chunk, "plan": _prepare_plan, "store": _prepare_store, "sample": _prepare_sample}[case["kind"]]
    return {**make(case, _generator(seed)), "case": case}


# ------------------------------------------------------------------------------------------------ the plain forms
def _chunk_plain(state):
    """Sequences padded to the longest chunk and the longest cache."""
    case, table, lengths, starts = state["case"], state["table"], state["lengths"], state["starts"]
    tokens, kv, group, dim = state["q"].shape
    n, most, cached = len(lengths), case["chunk"], table.shape[1] * case["page"]
    counts = starts[1:] - starts[:-1]
    i = torch.arange(most, device="cuda")[None, :]
    taken = i < counts[:, None]  # [n, most]
    place = torch.where(taken, starts[:-1, None] + i, 0)

    def keys_of(pages, new):  # [n, kv, cached (+ most), dim]
        found = pages[table.clamp(min=0)].float().reshape(n, cached, kv, dim)
        found = found if new is None else torch.cat([found, new.float()[place]], 1)
        return found.transpose(1, 2).contiguous()

    k, v = keys_of(state["k_pages"], state["k_new"]), keys_of(state["v_pages"], state["v_new"])
    j = torch.arange(cached, device="cuda")
    held = (j[None, :] < lengths[:, None])
    if state["k_new"] is None:
        position = (lengths - counts)[:, None] + i  # [n, most]
        where = j[None, :].expand(n, -1)
    else:
        position = lengths[:, None] + i
        where = torch.cat([j[None, :].expand(n, -1), position], 1)
        held = torch.cat([held, taken], 1)
    seen = held[:, None, :] & (where[:, None, :] <= position[:, :, None])  # [n, most, keys]
    if case["window"]:
        seen &= (where[:, None, :] > position[:, :, None] - case["window"]) | (where[:, None, :] < case["first"])
    q = (state["q"].float() * state["scale"])[place].reshape(n, most, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(n, kv, group * most, dim).contiguous()
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()).view(n, kv, group, most, -1)
    del k
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    sink = None if state["sinks"] is None else state["sinks"].float().view(1, kv, group, 1, 1)
    top = top if sink is None else torch.maximum(top, sink)
    top = torch.where(top == -math.inf, 0.0, top)
    weights = scores.sub_(top).exp_()
    total = weights.sum(-1, keepdim=True)
    total = total if sink is None else total + torch.exp(sink - top)
    mixed = torch.matmul(weights.view(n, kv, group * most, -1), v).view(n, kv, group, most, dim)
    result = torch.where(total > 0, mixed / total, 0.0).permute(0, 3, 1, 2, 4)
    return result[taken].to(state["q"].dtype)


def _plan_plain(state):
    lengths, counts, table, free, page = state["lengths"], state["counts"], state["table"], state["free"], state["case"]["page"]
    n, span = table.shape
    ends = counts.cumsum(0)
    starts = torch.cat([ends.new_zeros(1), ends])
    held = (lengths + page - 1) // page
    wanted = (lengths + counts + page - 1) // page - held
    before = wanted.cumsum(0) - wanted
    column = torch.arange(span, device="cuda")[None, :]
    fresh = (column >= held[:, None]) & (column < (held + wanted)[:, None])
    at = torch.where(fresh, state["cursor"] + before[:, None] + column - held[:, None], 0)
    table = torch.where(fresh, torch.where(at < len(free), free[at.clamp(max=len(free) - 1)], -1), table)
    t = torch.arange(state["tokens"], device="cuda")
    owner = torch.searchsorted(ends, t, right=True)
    valid = owner < n
    owner = owner.clamp(max=n - 1)
    position = lengths[owner] + t - starts[owner]
    slot = table[owner, (position // page).clamp(max=span - 1)] * page + position % page
    return {"table": table, "starts": starts, "slots": torch.where(valid, slot, -1), "positions": torch.where(valid, position, -1),
            "owners": torch.where(valid, owner, -1), "lengths": lengths + counts, "taken": state["cursor"] + wanted.sum()}


def _store_plain(state):
    stored = state["slots"] >= 0
    where = state["slots"][stored]
    state["keys"][:, where] = state["new_keys"][:, stored]
    state["values"][:, where] = state["new_values"][:, stored]
    return [state["keys"], state["values"]]


def _sample_plain(state):
    """In 64 bits: a token's mass may end next to the drawn place."""
    x, ids = torch.sort(state["logits"].float(), dim=1, descending=True, stable=True)
    rows, width = x.shape
    x, rank = x.double(), torch.arange(width, device="cuda")[None, :]
    temperature = state["temperature"].double()[:, None]
    weights = torch.exp((x - x[:, :1]) / torch.where(temperature > 0, temperature, 1.0))
    mass = weights.cumsum(1)
    kept = torch.full((rows, 1), width, dtype=torch.int64, device="cuda")
    if state["top_k"] is not None:
        k = state["top_k"][:, None]
        kept = torch.where((k > 0) & (k < width), k, kept)
        within = mass.gather(1, kept - 1)
        p = state["top_p"].double()[:, None]
        nucleus = (mass < p * within).sum(1, keepdim=True) + 1
        kept = torch.where(p < 1, torch.minimum(kept, nucleus), kept)
        floor = state["min_p"].double()[:, None]
        kept = torch.minimum(kept, (weights >= floor).sum(1, keepdim=True).clamp(min=1))
    total = mass.gather(1, kept - 1)
    chosen = ((mass <= state["uniform"].double()[:, None] * total) & (rank < kept - 1)).sum(1, keepdim=True)
    greedy = temperature <= 0
    chosen = torch.where(greedy, 0, chosen)
    logprobs = torch.where(greedy, 0.0, torch.log(weights.gather(1, chosen) / total))
    return {"ids": ids.gather(1, chosen)[:, 0], "logprobs": logprobs[:, 0].float()}


# ------------------------------------------------------------------------------------------------ the framework's calls
def _pointer(tensor):
    return None if tensor is None else tensor.data_ptr()


def _call(name, state, call):
    """One call of the C entry, in a workspace that a serving loop keeps."""
    from chroma_amd._src import native

    lib, error = native.library(), ctypes.create_string_buffer(256)
    if "workspace" not in state:
        need = getattr(lib, name + "_workspace")(ctypes.byref(call))
        state["workspace"] = torch.empty(max(1, need), dtype=torch.uint8, device="cuda")
    native.check(getattr(lib, name)(ctypes.byref(call), state["workspace"].data_ptr(), state["workspace"].numel(),
                                    torch.cuda.current_stream().cuda_stream, error, len(error)), error)


def _call_plain(name, call):
    """One call of a C entry that needs no workspace."""
    from chroma_amd._src import native

    error = ctypes.create_string_buffer(256)
    native.check(getattr(native.library(), name)(ctypes.byref(call), torch.cuda.current_stream().cuda_stream, error, len(error)), error)


def _chunk_own(state):
    from chroma_amd._src import native

    case, q = state["case"], state["q"]
    tokens, kv, group, dim = q.shape
    out = torch.empty_like(q)
    _call("chroma_hip_paged_chunk_attention", state, native.PagedChunk(
        q=q.data_ptr(), k_pages=state["k_pages"].data_ptr(), v_pages=state["v_pages"].data_ptr(), k_new=_pointer(state["k_new"]),
        v_new=_pointer(state["v_new"]), sinks=_pointer(state["sinks"]), table=state["table"].data_ptr(), lengths=state["lengths"].data_ptr(),
        starts=state["starts"].data_ptr(), out=out.data_ptr(), tokens=tokens, sequences=case["sequences"], kv_heads=kv, group=group, dim=dim,
        pages=state["k_pages"].shape[0], page_rows=case["page"], page_stride=case["page"] * kv * dim, row_stride=kv * dim, head_stride=dim,
        q_stride=kv * group * dim, new_stride=kv * dim, out_stride=kv * group * dim, table_stride=state["table"].shape[1],
        longest=case["longest"], window=case["window"], first=case["first"], scale=state["scale"],
        dtype=native.FLOAT32 if q.dtype == torch.float32 else native.BFLOAT16))
    return out


def _plan_own(state):
    from chroma_amd._src import native

    n, span = state["table"].shape
    made = {name: torch.empty(size, dtype=torch.int64, device="cuda") for name, size in
            (("starts", n + 1), ("slots", state["tokens"]), ("positions", state["tokens"]), ("owners", state["tokens"]), ("lengths", n), ("taken", 1))}
    _call_plain("chroma_hip_paged_plan", native.PagedPlan(
        lengths=state["lengths"].data_ptr(), counts=state["counts"].data_ptr(), free_pages=state["free"].data_ptr(),
        cursor=state["cursor"].data_ptr(), table=state["table"].data_ptr(), starts=made["starts"].data_ptr(), slots=made["slots"].data_ptr(),
        positions=made["positions"].data_ptr(), owners=made["owners"].data_ptr(), new_lengths=made["lengths"].data_ptr(),
        taken=made["taken"].data_ptr(), sequences=n, tokens=state["tokens"], pages=state["pages"], page_rows=state["case"]["page"], span=span,
        table_stride=span, free_count=len(state["free"])))
    return {"table": state["table"], **made}


def _store_own(state):
    from chroma_amd._src import native

    keys, new = state["keys"], state["new_keys"]
    layers, rows, row_bytes = keys.shape
    _call_plain("chroma_hip_cache_store", native.CacheStore(
        keys=keys.data_ptr(), values=state["values"].data_ptr(), new_keys=new.data_ptr(), new_values=state["new_values"].data_ptr(),
        slots=state["slots"].data_ptr(), layers=layers, rows=rows, count=new.shape[1], row_bytes=row_bytes, layer_pitch=rows * row_bytes,
        new_layer_pitch=new.stride(0), new_row_pitch=new.stride(1)))
    return [keys, state["values"]]


def _sample_own(state):
    from chroma_amd._src import native

    x = state["logits"]
    rows, width = x.shape
    ids, logprobs = torch.empty(rows, dtype=torch.int64, device="cuda"), torch.empty(rows, dtype=torch.float32, device="cuda")
    _call("chroma_hip_rows_sample", state, native.Sample(
        x=x.data_ptr(), rows=rows, width=width, x_stride=width, temperature=state["temperature"].data_ptr(), top_k=_pointer(state["top_k"]),
        top_p=_pointer(state["top_p"]), min_p=_pointer(state["min_p"]), uniform=state["uniform"].data_ptr(), ids=ids.data_ptr(),
        logprobs=logprobs.data_ptr(), dtype=native.FLOAT32 if x.dtype == torch.float32 else native.BFLOAT16))
    return {"ids": ids, "logprobs": logprobs}


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"chunk": _chunk_own, "plan": _plan_own, "store": _store_own, "sample": _sample_own}[kind](state)
    return {"chunk": _chunk_plain, "plan": _plan_plain, "store": _store_plain, "sample": _sample_plain}[kind](state)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["kind"] == "chunk":
        size = 4 if case["dtype"] == "f32" else 2
        n, longest = case["sequences"], case["longest"]
        heads, pairs, keys, tokens = case["kv_heads"] * case["group"], 0.0, 0.0, 0.0
        for b, new in enumerate(_counts(case)):
            if new == 0:
                continue
            cached = longest if b == 0 or case["mix"] == "even" else longest / 2  # the mean of what prepare() draws
            total = cached + new if case["fresh"] else max(cached, new)  # rows after the chunk
            seen = total - (new - 1) / 2  # by a token, on average
            if case["window"]:
                seen = min(seen, case["window"] + case["first"])
                total = min(total, case["window"] + case["first"] + new)
            pairs, keys, tokens = pairs + new * seen, keys + total, tokens + new
        return {"bytes": 2 * keys * case["kv_heads"] * case["dim"] * size + 2 * tokens * heads * case["dim"] * size + 8 * (keys / case["page"] + 2 * n),
                "flops": 4 * pairs * heads * case["dim"]}
    if case["kind"] == "plan":
        n, tokens = case["sequences"], case["sequences"] * (case["chunk"] if case["chunk"] == 1 else case["chunk"] / 2)
        return {"bytes": 32 * n + 16 * tokens / case["page"] + 24 * n * case["chunk"], "flops": 0}
    if case["kind"] == "store":
        return {"bytes": 4 * case["layers"] * case["tokens"] * case["row_bytes"] + 8 * case["tokens"], "flops": 0}
    elements = case["rows"] * case["width"]
    return {"bytes": elements * (4 if case["dtype"] == "f32" else 2) + 32 * case["rows"], "flops": 4 * elements}


# ------------------------------------------------------------------------------------------------ 64 bits, by the definitions
def _chunk_exact(state):
    """Sequence by sequence and head by head: the rows in order, each token's own, a softmax over them, the sum of their values."""
    case, page = state["case"], state["case"]["page"]
    tokens, kv, group, dim = state["q"].shape
    result = torch.zeros(tokens, kv, group, dim, dtype=torch.float64, device="cuda")
    starts = state["starts"].tolist()
    for b, length in enumerate(state["lengths"].tolist()):
        begin, end = starts[b], starts[b + 1]
        if begin == end:
            continue
        j = torch.arange(length, device="cuda")
        place = state["table"][b][j // page] * page + j % page
        now = torch.arange(end - begin, device="cuda") + (length if case["fresh"] else length - (end - begin))
        j = torch.arange(length + (end - begin if case["fresh"] else 0), device="cuda")
        hidden = j[None, :] > now[:, None]
        if case["window"]:
            hidden |= (now[:, None] - j[None, :] >= case["window"]) & (j[None, :] >= case["first"])
        for h in range(kv):
            k, v = (state[name].view(-1, kv, dim)[place, h].double() for name in ("k_pages", "v_pages"))
            if case["fresh"]:
                k, v = torch.cat([k, state["k_new"][begin:end, h].double()]), torch.cat([v, state["v_new"][begin:end, h].double()])
            for g in range(group):
                s = torch.mm(state["q"][begin:end, h, g].double(), k.t().contiguous()).mul_(state["scale"]).masked_fill_(hidden, -math.inf)
                if state["sinks"] is not None:
                    s = torch.cat([s, state["sinks"][h * group + g].double().expand(end - begin, 1)], 1)
                result[begin:end, h, g] = torch.mm(torch.softmax(s, 1)[:, : len(k)], v)
    return result


def _sample_exact(state):
    """Row by row: the logarithm of the chosen token's share. The token itself is a whole number."""
    x = state["logits"].double().cpu().numpy()
    settings = {name: None if state[name] is None else state[name].cpu().numpy() for name in ("temperature", "top_k", "top_p", "min_p", "uniform")}
    result = np.zeros(len(x))
    for r, row in enumerate(x):
        heat = float(settings["temperature"][r])
        if heat <= 0:
            continue
        share = np.exp((np.sort(row)[::-1] - row.max()) / heat)
        if settings["top_k"] is not None:
            k = int(settings["top_k"][r])
            share = share[:k] if k > 0 else share
            below = np.cumsum(share) < float(settings["top_p"][r]) * np.sum(share)
            within = share[: 1 + np.count_nonzero(below)] if settings["top_p"][r] < 1 else share
            least = max(1, np.count_nonzero(share >= float(settings["min_p"][r])))
            share = within[:least]
        upto = np.cumsum(share)
        chosen = min(np.searchsorted(upto, float(settings["uniform"][r]) * upto[-1], side="right"), len(share) - 1)
        result[r] = math.log(share[chosen] / upto[-1])
    return {"ids": None, "logprobs": torch.from_numpy(result)}


def exact(case, seed):
    if case["kind"] in ("plan", "store"):
        return None  # whole values: equal or not
    state = prepare(case, seed)
    return _chunk_exact(state) if case["kind"] == "chunk" else _sample_exact(state)
