"""What is measured of the learned projections in front of a table: the products grouped by source, the
low-rank adapters of many requests beside a shared projection, and the gradients of both.

Rows x [n, din] lie in segments: segment s holds rows [offsets[s], offsets[s + 1]); rows behind the last segment
belong to none and are left as they were.

  grouped            y_i = W[g(i)] x_i
  grouped_backward   dx_i = W[g(i)]^T dy_i,  dW[g] = sum over the rows of g of dy_i x_i^T
  adapted            y_i = W x_i + s[a(i)] B[a(i)] (A[a(i)] x_i),  a(i) the adapter of the row's request, -1 for none
  adapted_backward   dx_i = W^T dy_i + s A^T (B^T dy_i),  dA[a] = s sum of (B^T dy_i) x_i^T,  dB[a] = s sum of dy_i (A x_i)^T

With `own` false `run` computes them with elementary torch operations in 32 bits, rounded once; with `own` true it calls
the entry points of vectordb_amd.
"""
import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}


def _grouped(name, op, n, din, dout, sources, dtype, out, empty=0):
    return {"name": name, "op": op, "n": n, "din": din, "dout": dout, "segments": sources, "dtype": dtype, "out": out,
            "empty": empty, "pad": 0, "adapters": 0, "rank": 0}


def _adapted(name, op, n, din, dout, requests, adapters, rank, dtype, out, pad=0):
    return {"name": name, "op": op, "n": n, "din": din, "dout": dout, "segments": requests, "dtype": dtype, "out": out,
            "empty": 0, "pad": pad, "adapters": adapters, "rank": rank}


def listed():
    return [
        # a handful of merged queries embedded by three encoders, on the way into a 384-dimensional table
        _grouped("grouped_queries_f32", "grouped", 24, 384, 384, 3, "f32", "f32"),
        # one ingest batch of documents, images and code, one matrix for each encoder
        _grouped("grouped_ingest_bf16", "grouped", 8192, 768, 768, 8, "bf16", "bf16"),
        # bulk ingest: a wider encoder into a 768-dimensional table, rows leave as the fp32 that an insert takes
        _grouped("grouped_bulk_bf16", "grouped", 65536, 1024, 768, 5, "bf16", "f32", empty=1),
        # embeddings of odd widths (features appended to an embedding)
        _grouped("grouped_odd_f16", "grouped", 5003, 515, 387, 7, "f16", "f16", empty=2),
        # one step of fitting small fp32 maps
        _grouped("grouped_fit_f32", "grouped_backward", 1000, 384, 384, 4, "f32", "f32", empty=1),
        # one step of fitting the maps of eight encoders on a large batch
        _grouped("grouped_fit_bf16", "grouped_backward", 32768, 1024, 768, 8, "bf16", "f32"),
        # a single query with its tenant's adapter: latency
        _adapted("adapted_query_bf16", "adapted", 1, 768, 768, 1, 512, 16, "bf16", "f32"),
        # the single queries of 64 callers merged into one batch, nearly all with adapters of their own
        _adapted("adapted_callers_f32", "adapted", 64, 384, 384, 64, 100, 8, "f32", "f32"),
        # a batch of 1024 queries from 128 requests, padded at its end
        _adapted("adapted_batch_bf16", "adapted", 1024, 768, 768, 128, 96, 16, "bf16", "f32", pad=24),
        # stored embeddings of 48 tenants mapped again after a change of the embedding model
        _adapted("adapted_remap_f16", "adapted", 32768, 1024, 768, 48, 48, 64, "f16", "f16"),
        # a small step of fitting adapters in fp32
        _adapted("adapted_fit_f32", "adapted_backward", 256, 384, 384, 32, 20, 8, "f32", "f32"),
        # a large step of fitting adapters that several requests share
        _adapted("adapted_fit_bf16", "adapted_backward", 16384, 768, 768, 64, 24, 16, "bf16", "f32", pad=100),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["grouped", "grouped_backward", "adapted", "adapted_backward"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    out = rng.choice(["f32", dtype])
    odd = rng.random() < 0.3
    if odd:
        din, dout = rng.randint(33, 800), rng.randint(33, 800)
    else:
        din, dout = 8 * rng.randint(8, 192), 8 * rng.randint(8, 192)
    n = _log(rng, 1, 65536)
    # no dearer than the largest listed case, with fp32 and rows that are not aligned counted eight times
    most = 65536 * 1024 * 768 // (2 if op.endswith("backward") else 1) // (8 if odd or dtype == "f32" else 1)
    n = max(1, min(n, most // (din * dout)))
    if op.startswith("grouped"):
        return _grouped("", op, n, din, dout, rng.randint(1, 16), dtype, out, empty=rng.randint(0, 2))
    requests = max(1, min(n, _log(rng, 1, 256)))
    pad = rng.choice([0, 0, n // 20])
    return _adapted("", op, n, din, dout, requests, _log(rng, 1, 256), _log(rng, 1, 64), dtype, out, pad=pad)


def _segments(case, gen):
    """Ragged segment sizes over n - pad rows: a few long ones, many short ones, `empty` without rows."""
    s, rows = case["segments"], case["n"] - case["pad"]
    full = max(1, s - case["empty"])
    weight = torch.rand(full, generator=gen, dtype=torch.float64).add_(0.02).pow_(2)
    spare = max(0, rows - full)                     # every segment that is not empty starts from one row
    sizes = torch.floor(weight / weight.sum() * spare).long() + (1 if rows >= full else 0)
    sizes[int(torch.randint(full, (1,), generator=gen))] += rows - int(sizes.sum())
    at = torch.randperm(s, generator=gen)[:full].sort().values
    lens = torch.zeros(s, dtype=torch.int64)
    lens[at] = sizes
    return torch.cat([torch.zeros(1, dtype=torch.int64), lens.cumsum(0)])


def _inputs(case, seed):
    gen = torch.Generator().manual_seed(seed)
    offsets = _segments(case, gen)
    ids = None
    if case["adapters"]:
        order = torch.randperm(case["adapters"], generator=gen).int()
        ids = order[torch.arange(case["segments"]) % case["adapters"]].clone()
        ids[7::8] = -1                              # every eighth request has no adapter of its own
    dev = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPES[case["dtype"]]

    def normal(shape, scale):
        return (torch.randn(shape, generator=dev, device="cuda") * scale).to(dt)

    n, din, dout, r, count = case["n"], case["din"], case["dout"], case["rank"], case["adapters"]
    t = {"x": normal((n, din), din ** -0.5)}        # embeddings of norm one or so
    t["w"] = normal((1 if count else case["segments"], dout, din), din ** -0.5)
    if count:
        t["a"] = normal((count, r, din), din ** -0.5)
        t["b"] = normal((count, dout, r), 0.3 * r ** -0.5)
        t["scale"] = torch.rand(count, generator=dev, device="cuda") * 1.5 + 0.5
    if case["op"].endswith("backward"):
        t["dy"] = normal((n, dout), 1.0 / math.sqrt(n))
    return t, offsets, ids


def prepare(case, seed):
    t, offsets, ids = _inputs(case, seed)
    state = {"case": case, "t": t, "offsets": offsets.tolist(), "ids": ids.tolist() if ids is not None else None}
    if not own:
        return state
    from vectordb_amd.engine import Engine
    from vectordb_amd.projection import Projection
    engine = Engine(device=0)
    out = _DTYPES[case["out"]]
    proj = Projection(t["w"], a=t.get("a"), b=t.get("b"), scale=t.get("scale"), out_dtype=out)
    state.update(engine=engine, proj=proj, offsets_dev=offsets.cuda(), ids_dev=ids.cuda() if ids is not None else None)
    shapes = {"y": (case["n"], case["dout"])}
    if case["op"].endswith("backward"):
        shapes = {"dx": (case["n"], case["din"])}
        shapes.update({"dw": t["w"].shape} if not case["adapters"] else {"da": t["a"].shape, "db": t["b"].shape})
    state["outs"] = {k: torch.zeros(tuple(s), dtype=out, device="cuda") for k, s in shapes.items()}
    size = engine.projection_workspace_bytes(proj, case["n"], case["segments"], case["op"].endswith("backward"))
    state["ws"] = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
    state["ws_bytes"] = size
    return state


def _run_own(state):
    case, t, o, eng, proj = state["case"], state["t"], state["outs"], state["engine"], state["proj"]
    n, din, dout = case["n"], case["din"], case["dout"]
    stream = torch.cuda.current_stream().cuda_stream
    x, offsets = t["x"].data_ptr(), state["offsets_dev"].data_ptr()
    ws = (state["ws"].data_ptr(), state["ws_bytes"])
    if case["op"] == "grouped":
        eng.project_grouped_dev(proj, n, x, din, offsets, o["y"].data_ptr(), dout, stream=stream)
        return o["y"]
    if case["op"] == "grouped_backward":
        eng.project_grouped_backward_dev(proj, n, t["dy"].data_ptr(), dout, x, din, offsets, o["dx"].data_ptr(), din,
                                         o["dw"].data_ptr(), *ws, stream=stream)
        return o["dx"], o["dw"]
    ids = state["ids_dev"].data_ptr()
    if case["op"] == "adapted":
        eng.project_adapted_dev(proj, n, x, din, case["segments"], offsets, ids, o["y"].data_ptr(), dout, *ws, stream=stream)
        return o["y"]
    eng.project_adapted_backward_dev(proj, n, t["dy"].data_ptr(), dout, x, din, case["segments"], offsets, ids,
                                     o["dx"].data_ptr(), din, o["da"].data_ptr(), o["db"].data_ptr(), *ws, stream=stream)
    return o["dx"], o["da"], o["db"]


def _run_plain(state):
    case, t, off, ids = state["case"], state["t"], state["offsets"], state["ids"]
    out = _DTYPES[case["out"]]
    n, din, dout, segments = case["n"], case["din"], case["dout"], case["segments"]
    x, w = t["x"].float(), t["w"].float()
    f32 = dict(dtype=torch.float32, device="cuda")
    if case["op"] == "grouped":
        y = torch.zeros(n, dout, **f32)
        for g in range(segments):
            s, e = off[g], off[g + 1]
            if e > s:
                y[s:e] = x[s:e] @ w[g].T
        return y.to(out)
    if case["op"] == "grouped_backward":
        dy, dx, dw = t["dy"].float(), torch.zeros(n, din, **f32), torch.zeros(segments, dout, din, **f32)
        for g in range(segments):
            s, e = off[g], off[g + 1]
            if e > s:
                dx[s:e] = dy[s:e] @ w[g]
                dw[g] = dy[s:e].T @ x[s:e]
        return dx.to(out), dw.to(out)
    a, b, scale, last = t["a"].float(), t["b"].float(), t["scale"], off[-1]
    if case["op"] == "adapted":
        y = torch.zeros(n, dout, **f32)
        y[:last] = x[:last] @ w[0].T
        for i in range(segments):
            s, e, k = off[i], off[i + 1], ids[i]
            if e > s and k >= 0:
                y[s:e] += scale[k] * ((x[s:e] @ a[k].T) @ b[k].T)
        return y.to(out)
    dy, dx, da, db = t["dy"].float(), torch.zeros(n, din, **f32), torch.zeros_like(a), torch.zeros_like(b)
    dx[:last] = dy[:last] @ w[0]
    for i in range(segments):
        s, e, k = off[i], off[i + 1], ids[i]
        if e > s and k >= 0:
            g = scale[k] * (dy[s:e] @ b[k])
            h = scale[k] * (x[s:e] @ a[k].T)
            dx[s:e] += g @ a[k]
            da[k] += g.T @ x[s:e]
            db[k] += dy[s:e].T @ h
    return dx.to(out), da.to(out), db.to(out)


def run(state):
    return _run_own(state) if own else _run_plain(state)


def exact(case, seed):
    """The same outputs in 64 bits, by the adapter or source that each row has."""
    t, offsets, ids = _inputs(case, seed)
    d = {k: v.double() for k, v in t.items()}
    n, seg = case["n"], torch.searchsorted(offsets, torch.arange(case["n"]), right=True) - 1
    inside = (seg < case["segments"]).cuda()
    seg = seg.clamp(max=case["segments"] - 1)
    kind = (seg if ids is None else ids.long()[seg]).cuda()     # which matrix, or which adapter, a row goes through
    kind = torch.where(inside, kind, torch.full_like(kind, -1))
    rows_of = [(k, (kind == k).nonzero().squeeze(1)) for k in sorted(set(kind.tolist()) - {-1})]
    grad = case["op"].endswith("backward")
    src = d["dy"] if grad else d["x"]
    first = torch.zeros(n, case["din"] if grad else case["dout"], dtype=torch.float64, device="cuda")
    if ids is None:
        dw = torch.zeros_like(d["w"])
        for k, r in rows_of:
            m = d["w"][k]
            first[r] = src[r].mm(m if grad else m.t().contiguous())
            if grad:
                dw[k] = src[r].t().contiguous().mm(d["x"][r])
        return (first, dw) if grad else first
    m = d["w"][0]
    first[inside] = src[inside].mm(m if grad else m.t().contiguous())
    da, db = torch.zeros_like(d["a"]), torch.zeros_like(d["b"])
    for k, r in rows_of:
        full = d["scale"][k] * d["b"][k].mm(d["a"][k])          # the adapter as one matrix [dout, din]
        first[r] += src[r].mm(full if grad else full.t().contiguous())
        if grad:
            outer = d["scale"][k] * src[r].t().contiguous().mm(d["x"][r])       # gradient of that matrix
            da[k] = d["b"][k].t().contiguous().mm(outer)
            db[k] = outer.mm(d["a"][k].t().contiguous())
    return (first, da, db) if grad else first


def work(case):
    n, din, dout, r = case["n"] - case["pad"], case["din"], case["dout"], case["rank"]
    e, o = _BYTES[case["dtype"]], _BYTES[case["out"]]
    grad = case["op"].endswith("backward")
    if not case["adapters"]:
        full = max(1, case["segments"] - case["empty"])          # matrices that have rows
        weights = case["segments"] * dout * din
        if grad:
            return {"bytes": n * (din + dout) * e + full * dout * din * e + n * din * o + weights * o, "flops": 4 * n * din * dout}
        return {"bytes": n * din * e + full * dout * din * e + n * dout * o, "flops": 2 * n * din * dout}
    with_adapter = case["segments"] - case["segments"] // 8
    pair = min(with_adapter, case["adapters"]) * r * (din + dout)
    share = with_adapter / case["segments"]
    if grad:
        return {"bytes": n * (din + dout) * e + dout * din * e + pair * e + n * din * o + case["adapters"] * r * (din + dout) * o,
                "flops": int(2 * n * din * dout + 2 * n * share * r * (3 * din + 2 * dout))}
    return {"bytes": n * din * e + dout * din * e + pair * e + n * dout * o,
            "flops": int(2 * n * din * dout + 2 * n * share * r * (din + dout))}
