"""What is timed of the row operators: tables whose rows many entries share, and rows
sorted by group and back.

``run`` computes a case with elementary torch operations (``own = False``) or with the
package's operators (``own = True``); ``exact`` gives the same values in 64 bits.

    lookup    out[t] = scale * table[index[t]]
    gradient  grad_table[v] = scale * sum over index[t] = v of grad[t], and the rows touched
    group     the entries sorted by group, rows taken to their groups, and back with weights
    train     the same with the gradients of the rows, the group outputs and the weights

An index outside the table (or a group outside the groups) is an entry that is left out.
"""
import math

import torch

own = False

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
SIZES = {"float32": 4, "bfloat16": 2, "float16": 2}


def listed():
    f32, bf16, f16 = "float32", "bfloat16", "float16"
    return [
        # one row asked for, the latency of a call: the attributes of one picked Gaussian
        _table("lookup_one", "lookup", 1, 4096, 20, f32, "int64"),
        # the three colours of 300k Gaussians from a codebook of 4096 (rows of 12 bytes)
        _table("lookup_colours", "lookup", 300000, 4096, 3, f32, "int32"),
        # 1M Gaussians whose 59 attributes (position, shape, harmonics) come from 64k shared rows
        _table("lookup_attributes", "lookup", 1000000, 65536, 59, f32, "int32", skipped=0.01),
        # wide rows in 16 bits, sqrt(D) scaling, the table far larger than the caches
        _table("lookup_wide", "lookup", 16384, 131072, 2048, bf16, "int64", scale=math.sqrt(2048)),
        # a small batch: what a launch costs
        _table("gradient_small", "gradient", 512, 4096, 64, f32, "int64"),
        # the codebook's gradient from 300k Gaussians: tiny rows, so the order is what costs
        _table("gradient_colours", "gradient", 300000, 4096, 3, f32, "int32"),
        # 1M Gaussians on 64k rows of 59, an odd row of 236 bytes, some entries left out
        _table("gradient_attributes", "gradient", 1000000, 65536, 59, f32, "int32", skipped=0.01),
        # wide rows in 16 bits, most of the table untouched, a few rows hit very often
        _table("gradient_wide", "gradient", 32768, 131072, 1024, bf16, "int64", scale=32.0),
        # serving: 64 rows, each to 4 of 32 groups
        _group("group_small", "group", 64, 4, 32, 1024, bf16, f32),
        # 300k Gaussians sorted by their one depth plane of 3 with their 20 parameters, forward and backward
        _group("train_planes", "train", 300000, 1, 3, 20, f32, f32),
        # 100k Gaussians on 2 of 7 planes, odd 16-bit rows, some entries left out
        _group("train_soft", "train", 100003, 2, 7, 333, f16, f16, skipped=0.1),
        # wide rows to 4 of 64 groups, forward and backward
        _group("train_wide", "train", 16384, 4, 64, 2048, bf16, f32),
    ]


def _table(name, kind, entries, rows, width, dtype, index, scale=1.0, skipped=0.0):
    return {"name": name, "kind": kind, "entries": entries, "rows": rows, "width": width, "dtype": dtype,
            "index": index, "scale": scale, "skipped": skipped}


def _group(name, kind, entries, choices, groups, width, dtype, weights, skipped=0.0):
    return {"name": name, "kind": kind, "entries": entries, "choices": choices, "groups": groups, "width": width,
            "dtype": dtype, "weights": weights, "skipped": skipped}


def _spread(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    """A case of the listed ranges; at most 600 MB of rows in and out, so none costs more than the largest."""
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    skipped = rng.choice([0.0, 0.0, 0.02, 0.3])
    kind = rng.choice(["lookup", "gradient", "group", "train"])
    width = _spread(rng, 1, 2048)
    if kind in ("lookup", "gradient"):
        most = 300_000_000 // (width * SIZES[dtype])
        entries = _spread(rng, 1, max(1, min(1000000, most)))
        # a row's sum of thousands of entries stays within what 32 bits hold to their own accuracy
        rows = _spread(rng, max(2, entries // 1024), max(2, entries // 1024, min(262144, most)))
        case = _table("", kind, entries, rows, width, dtype, rng.choice(["int32", "int64"]),
                      rng.choice([1.0, 0.5, math.sqrt(width)]), skipped)
    else:
        choices = rng.randint(1, 8)
        most = 150_000_000 // (width * SIZES[dtype] * (choices + 1))
        entries = _spread(rng, 1, max(1, min(500000, most)))
        groups = _spread(rng, choices, 256)
        case = _group("", kind, entries, choices, groups, width, dtype, rng.choice([dtype, "float32"]), skipped)
    del case["name"]
    return case


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev, dtype, n, d = "cuda", TYPES[case["dtype"]], case["entries"], case["width"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    def left_out(index):
        if case["skipped"] > 0:
            index = torch.where(torch.rand(index.shape, generator=g, device=dev) < case["skipped"], -1, index)
        return index

    if case["kind"] in ("lookup", "gradient"):
        v = case["rows"]
        # rows are far from equally popular: density falls with the root of the row's (shuffled) rank
        rank = (torch.rand(n, generator=g, device=dev, dtype=torch.float64).square() * v).long().clamp_(max=v - 1)
        index = torch.randperm(v, generator=g, device=dev)[rank]
        s = {"case": case, "index": left_out(index).to(torch.int32 if case["index"] == "int32" else torch.int64)}
        if case["kind"] == "lookup":
            s["table"] = normal(v, d).to(dtype)
        else:
            s["grad"] = (normal(n, d) * 0.1).to(dtype)
        return s
    k = case["choices"]
    # the router: the k largest of the groups' logits, some groups liked more than others; a softmax over them
    logits = normal(n, case["groups"]) + normal(case["groups"])
    top, index = logits.topk(k, dim=1)
    s = {"case": case, "index": left_out(index).to(torch.int32), "x": normal(n, d).to(dtype),
         "y": normal(n * k, d).to(dtype), "weights": top.softmax(1).to(TYPES[case["weights"]])}
    if case["kind"] == "train":
        s["grad_rows"] = (normal(n, d) * 0.1).to(dtype)
        s["grad_groups"] = (normal(n * k, d) * 0.1).to(dtype)
        for name in ("x", "y", "weights"):
            s[name].requires_grad_(True)
    return s


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        from complex_valued_holographic_radiance_fields_b200 import rows as R
        if kind == "lookup":
            return R.table_lookup(state["table"], state["index"], case["scale"])
        if kind == "gradient":
            return R.table_gradient(state["grad"], state["index"], case["rows"], case["scale"])
        groups = R.group_rows(state["index"], case["groups"])
        xs = R.rows_to_groups(state["x"], groups)
        out = R.groups_to_rows(state["y"], groups, state["weights"])
        answer = {"order": groups.order, "slots": groups.slots, "offsets": groups.offsets, "xs": xs, "out": out}
        if kind == "train":
            answer["dx"], answer["dy"], answer["dw"] = torch.autograd.grad(
                (xs, out), (state["x"], state["y"], state["weights"]), (state["grad_groups"], state["grad_rows"]))
        return answer
    if kind == "lookup":
        return _plain_lookup(state["table"], state["index"], case["scale"])
    if kind == "gradient":
        return _plain_gradient(state["grad"], state["index"], case["rows"], case["scale"])
    with torch.no_grad():
        return _plain_groups(state, case)


def _plain_lookup(table, index, scale):
    inside = (index >= 0) & (index < table.shape[0])
    rows = table[torch.where(inside, index, 0)].float() * scale
    return torch.where(inside[:, None], rows, 0.0).to(table.dtype)


def _plain_gradient(grad, index, num_rows, scale):
    inside = (index >= 0) & (index < num_rows)
    at = torch.where(inside, index, num_rows)                   # one row more takes what is left out
    total = torch.zeros(num_rows + 1, grad.shape[1], device=grad.device)
    total.index_add_(0, at, grad.float())
    touched = torch.zeros(num_rows + 1, dtype=torch.uint8, device=grad.device)
    touched[at.long()] = 1
    return (total[:num_rows] * scale).to(grad.dtype), touched[:num_rows]


def _plain_groups(state, case):
    index, x, y, weights = state["index"], state["x"], state["y"], state["weights"]
    n, k = index.shape
    groups = case["groups"]
    inside = (index >= 0) & (index < groups)
    key = torch.where(inside, index, groups).reshape(-1)
    order = torch.sort(key, stable=True)[1]
    place = torch.empty_like(order)
    place[order] = torch.arange(n * k, device=order.device)
    place = place.view(n, k)
    count = torch.zeros(groups + 1, dtype=torch.int64, device=key.device)
    count.index_add_(0, key, torch.ones_like(key, dtype=torch.int64))
    offsets = torch.cat([count.new_zeros(1), count[:groups].cumsum(0)])
    used = (torch.arange(n * k, device=key.device) < offsets[-1])[:, None]
    kept = inside[:, :, None]
    xs = torch.where(used, x.float()[order // k], 0.0).to(x.dtype)
    rows = torch.where(kept, y.float()[place], 0.0)
    w = torch.where(inside, weights.float(), 0.0)
    out = (w[:, :, None] * rows).sum(1).to(y.dtype)
    answer = {"order": order.int(), "slots": torch.where(inside, place, -1).int(), "offsets": offsets.int(), "xs": xs,
              "out": out}
    if case["kind"] == "train":
        grad = state["grad_rows"].float()
        answer["dx"] = torch.where(kept, state["grad_groups"].float()[place], 0.0).sum(1).to(x.dtype)
        spread = grad[order // k] * w.reshape(-1)[order][:, None]
        answer["dy"] = torch.where(used, spread, 0.0).to(y.dtype)
        answer["dw"] = torch.where(inside, (grad[:, None, :] * rows).sum(2), 0.0).to(weights.dtype)
    return answer


def work(case):
    size, n, d = SIZES[case["dtype"]], case["entries"], case["width"]
    if case["kind"] == "lookup":
        read = n * (4 if case["index"] == "int32" else 8) + min(n, case["rows"]) * d * size
        return {"bytes": read + n * d * size, "flops": n * d}
    if case["kind"] == "gradient":
        read = n * (4 if case["index"] == "int32" else 8) + n * d * size
        return {"bytes": read + case["rows"] * (d * size + 1), "flops": n * d}
    k = case["choices"]
    entry = n * k * (4 + 4 + 4 + SIZES[case["weights"]])        # groups in; order and slots out; weights in
    row, grouped = n * d * size, n * k * d * size
    if case["kind"] == "group":
        return {"bytes": entry + 2 * row + 2 * grouped, "flops": 2 * n * k * d}
    return {"bytes": entry + n * k * SIZES[case["weights"]] + 4 * row + 4 * grouped, "flops": 6 * n * k * d}


def exact(case, seed):
    """The definitions, one choice at a time, in 64 bits; the whole numbers have no other value than run's."""
    s = prepare(case, seed)
    index = s["index"].long()
    if case["kind"] == "lookup":
        out = torch.zeros(case["entries"], case["width"], dtype=torch.float64, device=index.device)
        at = torch.nonzero((index >= 0) & (index < case["rows"]))[:, 0]
        out[at] = torch.index_select(s["table"], 0, index[at]).double().mul_(case["scale"])
        return out
    if case["kind"] == "gradient":
        at = torch.nonzero((index >= 0) & (index < case["rows"]))[:, 0]
        out = torch.zeros(case["rows"], case["width"], dtype=torch.float64, device=index.device)
        out.scatter_add_(0, index[at][:, None].expand(-1, case["width"]), s["grad"][at].double() * case["scale"])
        return out, None
    with torch.no_grad():
        return _exact_groups(case, s, index)


def _exact_groups(case, s, index):
    n, k = index.shape
    d, dev = case["width"], index.device
    # the place of an entry: all entries of lower groups, and those of its own group before it
    flat = index.reshape(-1)
    place = torch.full((n * k,), -1, dtype=torch.int64, device=dev)
    begin = 0
    for group in range(case["groups"]):
        at = torch.nonzero(flat == group)[:, 0]
        place[at] = begin + torch.arange(at.numel(), device=dev)
        begin += at.numel()
    place = place.view(n, k)

    def zeros(*shape):
        return torch.zeros(*shape, dtype=torch.float64, device=dev)

    answer = {"order": None, "slots": None, "offsets": None, "xs": zeros(n * k, d), "out": zeros(n, d)}
    train = case["kind"] == "train"
    if train:
        answer.update(dx=zeros(n, d), dy=zeros(n * k, d), dw=zeros(n, k))
    for j in range(k):
        row = torch.nonzero(place[:, j] >= 0)[:, 0]
        at = place[row, j]
        weight = s["weights"][row, j].double()[:, None]
        answer["xs"][at] = s["x"][row].double()
        answer["out"][row] += weight * s["y"][at].double()
        if train:
            grad = s["grad_rows"][row].double()
            answer["dx"][row] += s["grad_groups"][at].double()
            answer["dy"][at] = weight * grad
            answer["dw"][row, j] = torch.linalg.vecdot(grad, s["y"][at].double())
    return answer
