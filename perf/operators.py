"""Operators for fields made of several experts: samples sorted by the expert (block field) that each goes to and back with
weights, forward and gradient, and the linear layer in 8-bit integers with scales for each row and channel, dense and by expert.

Case keys: "op" names the operator.

  dispatch   expert ids [n][k] -> the plan (offsets, order, slot), and the rows of x in the experts' order
  combine    rows in the experts' order -> the weighted sum of each sample's k rows
  back       the gradient of both: of the combine (rows and weights) and of the dispatch
  linear_i8  x [m][n_in] brought to 8 bits row by row, times 8-bit weights [n_out][n_in], scales, bias, ReLU
  experts_i8 the same for rows sorted by expert, one weight matrix for each expert
"""
import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZES = {"f16": 2, "bf16": 2, "f32": 4}


def listed():
    return [
        # a handful of samples picked with the mouse, two blocks each, wide features: the latency of sort and gather
        dict(name="dispatch_few", op="dispatch", n=5, k=2, experts=8, d=256, dtype="bf16", outside=False),
        # a frame's samples as NerfCoordinate rows (position, dt, direction: 28 bytes), two overlapping blocks, some samples outside all
        dict(name="dispatch_coords", op="dispatch", n=1 << 20, k=2, experts=64, d=7, dtype="f32", outside=True),
        # the [n][4] network outputs of the same frame blended back
        dict(name="combine_outputs", op="combine", n=1 << 20, k=2, experts=64, d=4, dtype="f16", outside=True),
        # wide hidden rows, eight choices, an odd number of samples
        dict(name="combine_wide", op="combine", n=4099, k=8, experts=128, d=4096, dtype="bf16", outside=False),
        # a small training step in 32 bits, nothing aligned
        dict(name="back_odd", op="back", n=777, k=3, experts=5, d=333, dtype="f32", outside=True),
        # a large training step
        dict(name="back_wide", op="back", n=16384, k=2, experts=32, d=2048, dtype="f16", outside=False),
        # one row through a wide layer: bound by the weights
        dict(name="i8_one", op="linear_i8", m=1, n_in=4096, n_out=4096, dtype="bf16", relu=False, bias=False),
        # the hidden layer of the field's MLPs (64 wide) over half a frame's query budget
        dict(name="i8_field", op="linear_i8", m=1 << 20, n_in=64, n_out=64, dtype="f16", relu=True, bias=False),
        # a wide layer over many rows: bound by the matrix instructions
        dict(name="i8_wide", op="linear_i8", m=8192, n_in=4096, n_out=8192, dtype="bf16", relu=False, bias=True),
        # few rows spread over the experts
        dict(name="experts_few", op="experts_i8", m=48, experts=16, n_in=1024, n_out=2048, dtype="bf16", relu=True, bias=True, outside=False),
        # a grid of tiny fields: 32 encoded features to the 64-wide hidden layer
        dict(name="experts_fields", op="experts_i8", m=1 << 19, experts=512, n_in=32, n_out=64, dtype="f16", relu=True, bias=True, outside=True),
        # wide experts with many rows each
        dict(name="experts_wide", op="experts_i8", m=16384, experts=16, n_in=2048, n_out=4096, dtype="bf16", relu=True, bias=False, outside=False),
    ]


def _log(rng, lo, hi):
    v = int(lo * (hi / lo) ** rng.random() + 0.5)
    return min(hi, max(lo, v))


def draw(rng):
    op = rng.choice(["dispatch", "combine", "back", "linear_i8", "experts_i8"])
    dtype = rng.choice(["f16", "bf16", "f32"])
    size = SIZES[dtype]
    if op in ("dispatch", "combine", "back"):
        k = rng.randint(1, 8)
        n = _log(rng, 1, (1 << 20) // k)
        widest = min(4096, (100 << 20) // (n * k * size))
        d = _log(rng, 1, max(1, widest))
        if rng.random() < 0.4 and d >= 64:
            d -= d % 64
        return dict(op=op, n=n, k=k, experts=_log(rng, 1, 1024), d=d, dtype=dtype, outside=rng.random() < 0.5)
    experts = 1 if op == "linear_i8" else _log(rng, 1, 512)
    n_in = _log(rng, 16, 8192)
    n_out = _log(rng, 16, max(16, min(8192, (64 << 20) // (n_in * experts))))
    if rng.random() < 0.6:
        n_in, n_out = max(16, n_in - n_in % 16), max(16, n_out - n_out % 16)
    m = _log(rng, 1, max(1, min(1 << 20, (128 << 20) // (size * max(n_in, n_out)), (1 << 38) // (n_in * n_out))))
    c = dict(op=op, m=m, n_in=n_in, n_out=n_out, dtype=dtype, relu=rng.random() < 0.5, bias=rng.random() < 0.5)
    if op == "experts_i8":
        c.update(experts=experts, outside=rng.random() < 0.5)
    return c


def _expert_ids(case, gen, dev):
    """[n][k] ids, uneven over the experts; a share of the samples is outside (-1)."""
    n, k, e = case["n"], case["k"], case["experts"]
    first = (torch.rand(n, 1, generator=gen, device=dev) ** 1.5 * e).long().clamp_max(e - 1)
    step = torch.arange(k, device=dev)[None] * max(1, e // 7)
    ids = (first + step) % e
    if case["outside"]:
        ids = torch.where(torch.rand(n, k, generator=gen, device=dev) < 0.08, -1, ids)
    return ids.to(torch.int32)


def _plan(ids, e):
    """offsets [e + 1], order [n * k], slot [n][k]; the choices of one expert stay in their order."""
    key = torch.where((ids >= 0) & (ids < e), ids, e).reshape(-1)
    ordered, order = torch.sort(key, stable=True)
    offsets = torch.searchsorted(ordered, torch.arange(e + 1, device=ids.device, dtype=ordered.dtype))
    at = torch.arange(key.numel(), device=ids.device)
    slot = torch.empty_like(order)
    slot[order] = at
    slot = torch.where(key < e, slot, -1).reshape(ids.shape)
    order = torch.where(at < offsets[-1], order, -1)
    return offsets.to(torch.int32), order.to(torch.int32), slot.to(torch.int32)


def _rows(shape, gen, dev, dtype):
    x = torch.randn(shape, generator=gen, device=dev)
    return (x * torch.exp(0.5 * torch.randn(shape[0], 1, generator=gen, device=dev))).to(dtype)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    s = dict(case=case, dev=dev)
    if case["op"] in ("dispatch", "combine", "back"):
        n, k, d, e = case["n"], case["k"], case["d"], case["experts"]
        s["ids"] = _expert_ids(case, gen, dev)
        if case["op"] == "dispatch":
            s["x"] = _rows((n, d), gen, dev, dtype)
            s["rows"] = torch.zeros(n * k, d, device=dev, dtype=dtype)
            s["offsets"] = torch.empty(e + 1, device=dev, dtype=torch.int32)
            s["order"] = torch.empty(n * k, device=dev, dtype=torch.int32)
            s["slot"] = torch.empty(n, k, device=dev, dtype=torch.int32)
            return s
        s["offsets"], s["order"], s["slot"] = _plan(s["ids"], e)
        s["rows"] = _rows((n * k, d), gen, dev, dtype)
        s["weights"] = torch.softmax(torch.randn(n, k, generator=gen, device=dev), 1)
        s["y"] = torch.empty(n, d, device=dev, dtype=dtype)
        if case["op"] == "back":
            s["dy"] = _rows((n, d), gen, dev, dtype)
            s["dx_rows"] = _rows((n * k, d), gen, dev, dtype)
            s["drows"] = torch.zeros(n * k, d, device=dev, dtype=dtype)
            s["dweights"] = torch.empty(n, k, device=dev)
        return s
    m, n_in, n_out = case["m"], case["n_in"], case["n_out"]
    e = case.get("experts", 1)
    s["x"] = _rows((m, n_in), gen, dev, dtype)
    w = torch.randn(e, n_out, n_in, generator=gen, device=dev) * torch.exp(0.3 * torch.randn(e, n_out, 1, generator=gen, device=dev)) / n_in ** 0.5
    top = w.abs().amax(2)
    s["w"] = torch.round(w * (127.0 / top)[..., None]).to(torch.int8)
    s["w_scale"] = top / 127.0
    s["bias"] = torch.randn(e, n_out, generator=gen, device=dev) if case["bias"] else None
    s["y"] = torch.zeros(m, n_out, device=dev, dtype=dtype)
    if case["op"] == "experts_i8":
        ids = _expert_ids(dict(n=m, k=1, experts=e, outside=case["outside"]), gen, dev)
        s["offsets"] = _plan(ids, e)[0]
        s["most"] = int((s["offsets"][1:] - s["offsets"][:-1]).max())   # the plain form's padded batch
    return s


# ---- plain forms ----------------------------------------------------------------------------------------------------
def _dispatch(x, order, k, rows):
    got = x[order.clamp_min(0).long() // k]
    return torch.where((order >= 0)[:, None], got, rows)


def _combine(rows, weights, slot):
    kept = (slot >= 0)[..., None]
    got = torch.where(kept, rows[slot.clamp_min(0).long()].float(), 0.0)
    if weights is not None:
        got = got * torch.where(kept, weights[..., None], 0.0)
    return got.sum(1).to(rows.dtype)


def _combine_grad(dy, rows, weights, slot, order, drows):
    k = slot.shape[1]
    at = order.clamp_min(0).long()
    g = dy.float()
    d = g[at // k] * weights.reshape(-1)[at][:, None]
    d = torch.where((order >= 0)[:, None], d.to(rows.dtype), drows)
    got = torch.where((slot >= 0)[..., None], rows[slot.clamp_min(0).long()].float(), 0.0)
    return d, (got * g[:, None]).sum(2)


def _to_i8(x):
    """A row's values as round(127 x / a), a the row's largest, with the scale a / 127; the rounding's border needs 64 bits."""
    a = x.float().abs().amax(1, keepdim=True).clamp_min(2.0 ** -100)
    q = torch.round(x.double() * 127.0 / a.double())
    return q.float(), a / 127.0


def _finish(acc, scale, w_scale, bias, relu, dtype):
    y = acc * scale * w_scale
    if bias is not None:
        y = y + bias
    return (torch.relu(y) if relu else y).to(dtype)


def _linear(s):
    c = s["case"]
    q, scale = _to_i8(s["x"])
    acc = q @ s["w"][0].float().t()
    return _finish(acc, scale, s["w_scale"], s["bias"], c["relu"], s["x"].dtype)


def _linear_experts(s):
    c, offsets = s["case"], s["offsets"].long()
    q, scale = _to_i8(s["x"])
    at = torch.arange(c["m"], device=s["dev"])
    e = torch.searchsorted(offsets[1:].contiguous(), at, right=True).clamp_max(c["experts"] - 1)
    batch = offsets[:-1, None] + torch.arange(s["most"], device=s["dev"])
    acc = torch.bmm(q[batch.clamp_max(c["m"] - 1)], s["w"].float().transpose(1, 2).contiguous())
    acc = acc[e, (at - offsets[e]).clamp_max(s["most"] - 1)]
    y = _finish(acc, scale, s["w_scale"][e], s["bias"][e] if c["bias"] else None, c["relu"], s["x"].dtype)
    return torch.where((at < offsets[-1])[:, None], y, s["y"])


# ---- the framework's operators --------------------------------------------------------------------------------------
_held = {}


def _testbed():
    if "testbed" not in _held:
        import synerfgine_amd as sng
        _held["testbed"] = sng.Testbed(torch.cuda.current_device())
        _held["types"] = {torch.float16: sng.F16, torch.bfloat16: sng.BF16, torch.float32: sng.F32}
    return _held["testbed"], _held["types"]


def _workspace(s, size):
    if size and ("workspace" not in s or s["workspace"].numel() < size):
        s["workspace"] = torch.empty(size, device=s["dev"], dtype=torch.uint8)
    return (s["workspace"].data_ptr() if size else 0), size


def _run_own(s):
    tb, types = _testbed()
    c = s["case"]
    stream = torch.cuda.current_stream().cuda_stream
    t = types[DTYPES[c["dtype"]]]
    if c["op"] == "dispatch":
        n, k, d = c["n"], c["k"], c["d"]
        ws, ws_bytes = _workspace(s, tb.expert_sort_workspace(n, k, c["experts"]))
        tb.expert_sort(s["ids"].data_ptr(), n, k, c["experts"], s["offsets"].data_ptr(), s["order"].data_ptr(), s["slot"].data_ptr(), ws, ws_bytes, stream)
        tb.expert_dispatch(s["x"].data_ptr(), t, d, d, s["order"].data_ptr(), s["slot"].data_ptr(), n, k, s["rows"].data_ptr(), d, stream)
        return s["offsets"], s["order"], s["slot"], s["rows"]
    if c["op"] == "combine":
        n, k, d = c["n"], c["k"], c["d"]
        tb.expert_combine(s["rows"].data_ptr(), t, d, d, s["weights"].data_ptr(), s["slot"].data_ptr(), n, k, s["y"].data_ptr(), d, stream)
        return s["y"]
    if c["op"] == "back":
        n, k, d = c["n"], c["k"], c["d"]
        tb.expert_combine_backward(s["dy"].data_ptr(), d, s["rows"].data_ptr(), d, t, d, s["weights"].data_ptr(), s["slot"].data_ptr(), n, k,
                                   s["drows"].data_ptr(), d, s["dweights"].data_ptr(), stream)
        tb.expert_dispatch_backward(s["dx_rows"].data_ptr(), t, d, d, s["slot"].data_ptr(), n, k, s["y"].data_ptr(), d, stream)
        return s["drows"], s["dweights"], s["y"]
    m, n_in, n_out, e = c["m"], c["n_in"], c["n_out"], c.get("experts", 1)
    ws, ws_bytes = _workspace(s, tb.linear_i8_workspace(m, n_in, n_out, t, e))
    tb.linear_i8(s["x"].data_ptr(), t, m, n_in, n_in, s["w"].data_ptr(), n_in, s["w_scale"].data_ptr(), n_out, s["y"].data_ptr(), t, n_out,
                 d_bias=s["bias"].data_ptr() if c["bias"] else 0, relu=c["relu"], d_offsets=s["offsets"].data_ptr() if "experts" in c else 0, n_experts=e,
                 d_workspace=ws, workspace_bytes=ws_bytes, stream=stream)
    return s["y"]


def run(state):
    if own:
        return _run_own(state)
    s, c = state, state["case"]
    if c["op"] == "dispatch":
        offsets, order, slot = _plan(s["ids"], c["experts"])
        return offsets, order, slot, _dispatch(s["x"], order, c["k"], s["rows"])
    if c["op"] == "combine":
        return _combine(s["rows"], s["weights"], s["slot"])
    if c["op"] == "back":
        d, dw = _combine_grad(s["dy"], s["rows"], s["weights"], s["slot"], s["order"], s["drows"])
        return d, dw, _combine(s["dx_rows"], None, s["slot"])
    return _linear(s) if c["op"] == "linear_i8" else _linear_experts(s)


def work(case):
    size = SIZES[case["dtype"]]
    if case["op"] in ("dispatch", "combine", "back"):
        n, k, d = case["n"], case["k"], case["d"]
        row, all_rows, choices = n * d * size, n * k * d * size, 4 * n * k
        if case["op"] == "dispatch":
            return {"bytes": row + all_rows + 3 * choices + 4 * case["experts"], "flops": 0}
        if case["op"] == "combine":
            return {"bytes": row + all_rows + 2 * choices, "flops": 2 * n * k * d}
        return {"bytes": 2 * row + 3 * all_rows + 3 * choices, "flops": 4 * n * k * d}
    m, n_in, n_out, e = case["m"], case["n_in"], case["n_out"], case.get("experts", 1)
    return {"bytes": m * (n_in + n_out) * size + e * n_out * (n_in + 4 + 4 * case["bias"]), "flops": 2 * m * n_in * n_out}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    k = case.get("k", 1)
    if case["op"] == "dispatch":
        ids = s["ids"].reshape(-1)
        rows = s["rows"].double()
        kept = [torch.nonzero(ids == e).reshape(-1) for e in range(case["experts"])]
        at = torch.cat(kept)
        rows[:at.numel()] = s["x"].double()[torch.div(at, k, rounding_mode="floor")]
        return None, None, None, rows
    if case["op"] in ("combine", "back"):
        def total(rows, weights):
            y = torch.zeros(case["n"], case["d"], device=s["dev"], dtype=torch.float64)
            for j in range(k):
                t = torch.nonzero(s["slot"][:, j] >= 0).reshape(-1)
                part = rows[s["slot"][t, j].long()].double()
                y[t] += part if weights is None else part * weights[t, j, None].double()
            return y
        if case["op"] == "combine":
            return total(s["rows"], s["weights"])
        d, dw = s["drows"].double(), torch.zeros(case["n"], k, device=s["dev"], dtype=torch.float64)
        for j in range(k):
            t = torch.nonzero(s["slot"][:, j] >= 0).reshape(-1)
            p = s["slot"][t, j].long()
            g = s["dy"][t].double()
            d[p] = g * s["weights"][t, j, None].double()
            dw[t, j] = torch.linalg.vecdot(g, s["rows"][p].double())
        return d, dw, total(s["dx_rows"], None)
    y = s["y"].double()
    ends = s["offsets"].tolist() if case["op"] == "experts_i8" else [0, case["m"]]
    for e, (b, t) in enumerate(zip(ends[:-1], ends[1:])):
        if t == b:
            continue
        x = s["x"][b:t].double()
        a = torch.maximum(x.max(1).values, -x.min(1).values).clamp_min(2.0 ** -100)
        q = torch.round(127.0 * x / a[:, None])
        v = torch.matmul(q, s["w"][e].double().t()) * torch.outer(a / 127.0, s["w_scale"][e].double())
        v = v + s["bias"][e].double() if case["bias"] else v
        y[b:t] = v.clamp_min(0.0) if case["relu"] else v
    return y
