"""The operators on scores and on routed rows, as cases that can be timed: their inputs, one pass through each, in plain
torch operations and through the library's entry points, and the bytes and operations that a pass cannot do without.

  adjust    scores [rows, classes] with penalties for the classes that a row has shown already, biases, and masks of the
            classes that it may have
  top       the best classes of every row with their softmax weights (and the scores' gradient)
  dispatch  rows sorted by the expert (model) that each goes to
  combine   the experts' rows brought back and added with weights (and the gradients of rows and weights)
"""
import torch

own = False  # True: the library's kernels; False: the plain form

DEVICE = "cuda:0"
TYPES = {"f64": torch.float64, "f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f64": 0, "f32": 1, "f16": 2, "bf16": 3}  # the library's names of the types
SIZES = {"f64": 8, "f32": 4, "f16": 2, "bf16": 2}


def _adjust(**k):
    return dict(dict(op="adjust", type="bf16", rows=1, classes=10, pad=0, history=0, prompt=0.5, biases=0, class_bias=False,
                     masks=0, masked_rows=1.0, density=0.5), **k)


def _top(**k):
    return dict(dict(op="top", type="f32", rows=1, classes=8, pad=0, count=2, among=True, closed=0.0, backward=False), **k)


def _dispatch(**k):
    return dict(dict(op="dispatch", type="bf16", rows=1, per_row=2, width=8, experts=8, dropped=0.0, skew=1.0), **k)


def _combine(**k):
    return dict(dict(op="combine", type="bf16", rows=1, per_row=2, width=8, experts=8, dropped=0.0, skew=1.0, weighted=True,
                     backward=False), **k)


def listed():
    return [
        # one row that is answered step by step: an odd number of classes, a short history, a few biases, a grammar's mask
        dict(_adjust(type="f16", rows=1, classes=50021, history=200, biases=8, masks=1), name="adjust_one_row"),
        # a server's batch: long histories, biases on request, masks for half of the rows; rows padded to whole lines
        dict(_adjust(type="bf16", rows=64, classes=131000, pad=72, history=3000, biases=20, masks=16, masked_rows=0.5,
                     density=0.1), name="adjust_serving"),
        # a large batch of single-precision scores, penalties over very long histories
        dict(_adjust(type="f32", rows=384, classes=100003, history=12000), name="adjust_long_history"),
        # raw values of a ten-class model: priors shifted, classes that the document has had made less likely, one mask per document
        dict(_adjust(type="f64", rows=2_000_000, classes=10, history=2, prompt=0.0, class_bias=True, masks=2_000_000,
                     density=0.8), name="adjust_ten_classes"),
        # the gate of a few rows that wait for an answer
        dict(_top(type="f32", rows=5, classes=64, count=2), name="top_few_rows"),
        # the gate of a training step, some experts off, and its gradient
        dict(_top(type="bf16", rows=131072, classes=128, count=8, closed=0.05, backward=True), name="top_training"),
        # the three likeliest of ten classes and their probabilities, for every document of a table
        dict(_top(type="f64", rows=2_000_000, classes=10, count=3, among=False), name="top_ten_classes"),
        # a few rows to their experts
        dict(_dispatch(type="bf16", rows=7, per_row=2, width=4096, experts=16), name="dispatch_few_rows"),
        # documents sorted by the model of their segment; some have none
        dict(_dispatch(type="f32", rows=1_000_003, per_row=1, width=200, experts=37, dropped=0.01, skew=2.0),
             name="dispatch_documents"),
        # the rows of a training step to four experts each
        dict(_dispatch(type="bf16", rows=16384, per_row=4, width=4096, experts=64), name="dispatch_training"),
        # two models' ten raw values for each document, mixed
        dict(_combine(type="f64", rows=1_000_003, per_row=2, width=10, experts=5), name="combine_documents"),
        # the experts' rows of a training step back, with the gradients of rows and weights
        dict(_combine(type="bf16", rows=16384, per_row=4, width=4096, experts=64, dropped=0.02, backward=True),
             name="combine_training"),
    ]


def draw(rng):
    """One more case of the ranges that the listed ones stand for."""
    def log_int(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))

    family = rng.choice(["vocabulary", "vocabulary", "classes", "gate", "gate_training", "top_classes", "dispatch", "documents",
                         "combine", "combine_training", "mixture"])
    if family == "vocabulary":
        classes = log_int(2000, 131072)
        rows = log_int(1, max(1, min(384, 32_000_000 // classes)))
        masks = rng.choice([0, 1, rows])
        return _adjust(type=rng.choice(["f32", "f16", "bf16"]), rows=rows, classes=classes, pad=rng.choice([0, 0, 5, 64]),
                       history=rng.choice([0, log_int(1, 12000)]), prompt=rng.random(), biases=rng.choice([0, log_int(1, 300)]),
                       class_bias=rng.random() < 0.25, masks=masks, masked_rows=rng.choice([0.3, 1.0]),
                       density=rng.choice([0.001, 0.1, 0.9]))
    if family == "classes":
        classes = log_int(2, 1000)
        rows = log_int(100, 16_000_000 // classes)
        return _adjust(type=rng.choice(["f64", "f64", "f32"]), rows=rows, classes=classes, pad=rng.choice([0, 0, 3]),
                       history=rng.choice([0, 1, 5]), prompt=rng.random(), biases=rng.choice([0, 2]),
                       class_bias=rng.random() < 0.5, masks=rng.choice([0, 1, rows]), density=rng.choice([0.3, 0.8]))
    if family in ("gate", "gate_training"):
        classes = log_int(4, 512)
        rows = log_int(1, 512) if family == "gate" else log_int(1000, 16_000_000 // classes)
        return _top(type=rng.choice(["f32", "bf16", "f16"]), rows=rows, classes=classes, pad=rng.choice([0, 0, 4]),
                    count=rng.randint(1, min(8, classes)), among=rng.random() < 0.6, closed=rng.choice([0.0, 0.3]),
                    backward=family == "gate_training")
    if family == "top_classes":
        classes = log_int(3, 1000)
        return _top(type="f64", rows=log_int(100, 16_000_000 // classes), classes=classes, count=rng.randint(1, min(5, classes)),
                    among=False)
    experts, dropped, skew = log_int(2, 256), rng.choice([0.0, 0.05]), rng.choice([0.0, 1.0, 3.0])
    per_row = rng.randint(1, min(8, experts))
    if family in ("documents", "mixture"):
        experts, per_row = log_int(2, 100), rng.randint(1, 2)
        if family == "mixture":
            return _combine(type="f64", rows=log_int(1000, 1_000_000), per_row=per_row, width=rng.randint(1, 10), experts=experts,
                            dropped=dropped, skew=skew, weighted=rng.random() < 0.7)
        return _dispatch(type="f32", rows=log_int(1000, 500_000), per_row=per_row, width=rng.randint(5, 200), experts=experts,
                         dropped=dropped, skew=skew)
    width = log_int(64, 8192)
    rows = log_int(1, max(1, min(65536, 150_000_000 // (width * per_row))))
    kind = rng.choice(["f32", "bf16", "f16"])
    if family == "dispatch":
        return _dispatch(type=kind, rows=rows, per_row=per_row, width=width, experts=experts, dropped=dropped, skew=skew)
    return _combine(type=kind, rows=rows, per_row=per_row, width=width, experts=experts, dropped=dropped, skew=skew,
                    weighted=rng.random() < 0.8, backward=family == "combine_training")


# ---- inputs

def _offsets(lengths):
    return torch.cat([torch.zeros(1, dtype=torch.int64, device=DEVICE), torch.cumsum(lengths, 0)])


def _padded(values, pad):
    """The values as the first columns of a wider table."""
    if not pad:
        return values
    wide = torch.full((values.shape[0], values.shape[1] + pad), float("nan"), dtype=values.dtype, device=DEVICE)
    wide[:, :values.shape[1]] = values
    return wide[:, :values.shape[1]]


def _prepare_adjust(case, rand, randn):
    rows, classes, kind = case["rows"], case["classes"], TYPES[case["type"]]
    s = dict(scores=_padded((randn(rows, classes, kind if kind == torch.float64 else torch.float32) * 4).to(kind), case["pad"]))
    if case["history"]:
        # lengths around the mean, none for some rows; classes as they come in earnest, few of them often
        lengths = (rand(rows) * 2 * case["history"]).round().to(torch.int64)
        s["history_offsets"] = _offsets(lengths)
        s["history"] = (classes * rand(int(s["history_offsets"][-1])) ** 3).to(torch.int32).clamp_(max=classes - 1)
        s["prompts"] = (rand(rows) * 2 * case["prompt"] * lengths).to(torch.int32)
        s["repetition"], s["frequency"], s["presence"] = 1 + 0.5 * rand(rows), 0.5 * rand(rows), 0.5 * rand(rows)
    if case["biases"]:
        s["bias_offsets"] = _offsets((rand(rows) * 2 * case["biases"]).round().to(torch.int64))
        count = int(s["bias_offsets"][-1])
        s["bias_classes"] = (classes * rand(count)).to(torch.int32).clamp_(max=classes - 1)
        s["bias_values"] = randn(count) * 5
    if case["class_bias"]:
        s["class_bias"] = randn(classes)
    if case["masks"]:
        words = (classes + 31) // 32
        bits = torch.zeros(case["masks"], words, dtype=torch.int32, device=DEVICE)
        for b in range(32):
            bits |= (rand(case["masks"] * words) < case["density"]).view(-1, words).to(torch.int32) << b
        s["allowed"] = bits
        # which mask a row has: its own where there is one for each, else one of a few; -1: none
        mask = torch.arange(rows, device=DEVICE) if case["masks"] == rows else (rand(rows) * case["masks"]).long().clamp_(max=case["masks"] - 1)
        s["allowed_rows"] = torch.where(rand(rows) < case["masked_rows"], mask, -1).to(torch.int32)
    return s


def _prepare_top(case, rand, randn):
    rows, classes, kind = case["rows"], case["classes"], TYPES[case["type"]]
    scores = randn(rows, classes, kind if kind == torch.float64 else torch.float32) * 2
    if case["closed"]:
        scores[rand(rows * classes).view(rows, classes) < case["closed"]] = float("-inf")
    s = dict(scores=_padded(scores.to(kind), case["pad"]))
    if case["backward"]:
        s["gradients"] = randn(rows, case["count"])
    return s


def _routes(case, rand):
    """Experts of every row, all different, some of them much more asked for than others; -1: none."""
    rows, per_row, experts = case["rows"], case["per_row"], case["experts"]
    liked = rand(experts) * case["skew"]
    ids = torch.topk(liked + rand(rows * experts).view(rows, experts), per_row, dim=1).indices.to(torch.int32)
    if case["dropped"]:
        ids[rand(rows * per_row).view(rows, per_row) < case["dropped"]] = -1
    return ids


def _places(ids, experts):
    """Where each slot goes when the slots are sorted by expert (-1: nowhere), and where each expert's slots begin."""
    flat = ids.reshape(-1).to(torch.int64)
    valid = (flat >= 0) & (flat < experts)
    order = torch.sort(torch.where(valid, flat, experts), stable=True).indices
    places = torch.empty_like(order)
    places[order] = torch.arange(order.numel(), device=order.device)
    counts = torch.zeros(experts + 1, dtype=torch.int64, device=order.device)
    counts.index_add_(0, torch.where(valid, flat + 1, 0), valid.to(torch.int64))
    return torch.where(valid, places, -1).to(torch.int32).view(ids.shape), torch.cumsum(counts, 0).to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)

    def rand(n):
        return torch.rand(n, generator=g, device=DEVICE)

    def randn(*shape_and_type):
        kind = shape_and_type[-1] if isinstance(shape_and_type[-1], torch.dtype) else torch.float32
        shape = [n for n in shape_and_type if not isinstance(n, torch.dtype)]
        return torch.randn(shape, generator=g, device=DEVICE, dtype=kind)

    kind, op = TYPES[case["type"]], case["op"]
    if op == "adjust":
        s = _prepare_adjust(case, rand, randn)
    elif op == "top":
        s = _prepare_top(case, rand, randn)
    else:
        slots, width = case["rows"] * case["per_row"], case["width"]
        draw_type = kind if kind == torch.float64 else torch.float32
        ids = _routes(case, rand)
        if op == "dispatch":
            # the buffer of sorted rows is the program's; rows behind the last one that is sent stay as they are
            s = dict(ids=ids, source=randn(case["rows"], width, draw_type).to(kind), sorted=torch.zeros(slots, width, dtype=kind, device=DEVICE))
        else:
            s = dict(places=_places(ids, case["experts"])[0], sorted=randn(slots, width, draw_type).to(kind))
            if case["weighted"]:
                s["weights"] = torch.softmax(randn(case["rows"], case["per_row"], draw_type), 1)
            if case["backward"]:
                s["gradients"] = randn(case["rows"], width, draw_type).to(kind)
                s["sorted_gradients"] = torch.zeros(slots, width, dtype=kind, device=DEVICE)
    s["case"] = case
    return s


# ---- the plain form

def _plain_adjust(s):
    scores = s["scores"]
    rows, classes = scores.shape
    acc = torch.float64 if scores.dtype == torch.float64 else torch.float32
    x = scores.to(acc)
    if "history" in s:
        entry = torch.arange(s["history"].numel(), device=DEVICE)
        row = torch.searchsorted(s["history_offsets"], entry, right=True) - 1
        flat = row * classes + s["history"]
        seen = torch.zeros(rows * classes, dtype=torch.bool, device=DEVICE).index_fill_(0, flat, True).view(rows, classes)
        generated = (entry - s["history_offsets"][row] >= s["prompts"][row]).to(torch.int32)
        counts = torch.zeros(rows * classes, dtype=torch.int32, device=DEVICE).index_add_(0, flat, generated).view(rows, classes)
        repetition, frequency, presence = (s[k].to(acc)[:, None] for k in ("repetition", "frequency", "presence"))
        x = torch.where(seen, torch.where(x > 0, x / repetition, x * repetition), x)
        x = x - frequency * counts - torch.where(counts > 0, presence, 0)
    if "class_bias" in s:
        x = x + s["class_bias"].to(acc)
    if "bias_classes" in s and s["bias_classes"].numel():
        entry = torch.arange(s["bias_classes"].numel(), device=DEVICE)
        row = torch.searchsorted(s["bias_offsets"], entry, right=True) - 1
        last = torch.full((rows * classes,), -1, dtype=torch.int64, device=DEVICE)
        last = last.scatter_reduce(0, row * classes + s["bias_classes"], entry, "amax").view(rows, classes)
        x = x + torch.where(last >= 0, s["bias_values"].to(acc)[last.clamp(min=0)], 0)
    if "allowed" in s:
        c = torch.arange(classes, device=DEVICE)
        mask = s["allowed_rows"].to(torch.int64)
        bits = (s["allowed"][mask.clamp(min=0)][:, c >> 5] >> (c & 31).to(torch.int32)) & 1
        x = torch.where((mask < 0)[:, None] | (bits == 1), x, float("-inf"))
    return x.to(scores.dtype)


def _plain_top(s):
    case, scores = s["case"], s["scores"]
    acc = torch.float64 if scores.dtype == torch.float64 else torch.float32
    x = scores.to(acc)
    ordered, indexes = torch.sort(x, dim=1, descending=True, stable=True)
    chosen, indexes = ordered[:, :case["count"]], indexes[:, :case["count"]]
    best = ordered[:, :1]
    some = best > float("-inf")
    e_all = torch.where(some, torch.exp(x - best), 0)
    e = torch.where(some, torch.exp(chosen - best), 0)
    total = (e if case["among"] else e_all).sum(1, keepdim=True)
    weights = torch.where(some, e / total, 0)
    indexes = torch.where(chosen > float("-inf"), indexes, -1)
    out = [indexes.to(torch.int32), weights]
    if case["backward"]:
        g = s["gradients"].to(acc)
        mean = (g * weights).sum(1, keepdim=True)
        dx = torch.zeros_like(x) if case["among"] else torch.where(some, -(e_all / total) * mean, 0)
        part = weights * (g - mean) if case["among"] else weights * g
        dx.scatter_add_(1, indexes.clamp(min=0), torch.where(indexes >= 0, part, 0))
        out.append(dx.to(scores.dtype))
    return out


def _plain_dispatch(s):
    case = s["case"]
    places, offsets = _places(s["ids"], case["experts"])
    flat = places.view(-1).to(torch.int64)
    slots = torch.nonzero(flat >= 0).view(-1)
    s["sorted"][flat[slots]] = s["source"][slots // case["per_row"]]
    return [places, offsets, s["sorted"]]


def _plain_combine(s):
    case, rows = s["case"], s["sorted"]
    acc = torch.float64 if rows.dtype == torch.float64 else torch.float32
    places = s["places"].to(torch.int64)
    there = places >= 0
    picked = torch.where(there[:, :, None], rows[places.clamp(min=0)].to(acc), 0)
    weights = torch.where(there, s["weights"].to(acc), 0) if case["weighted"] else there.to(acc)
    out = [(picked * weights[:, :, None]).sum(1).to(rows.dtype)]
    if case["backward"]:
        g = s["gradients"].to(acc)
        spread = (weights[:, :, None] * g[:, None, :]).to(rows.dtype)
        s["sorted_gradients"][places[there]] = spread[there]
        out.append(s["sorted_gradients"])
        if case["weighted"]:
            out.append((picked * g[:, None, :]).sum(2))
    return out


# ---- the library's calls

def _at(s, name):
    return s[name].data_ptr() if name in s else 0


def _own_adjust(s, cb, code, stream):
    scores = s["scores"]
    rows, classes = scores.shape
    result = torch.empty(rows, classes, dtype=scores.dtype, device=DEVICE)
    adjustment = cb.score_adjustment(
        history_offsets_ptr=_at(s, "history_offsets"), history_ptr=_at(s, "history"), history_count=s["history"].numel() if "history" in s else 0,
        prompt_lengths_ptr=_at(s, "prompts"), repetition_ptr=_at(s, "repetition"), frequency_ptr=_at(s, "frequency"), presence_ptr=_at(s, "presence"),
        class_bias_ptr=_at(s, "class_bias"), bias_offsets_ptr=_at(s, "bias_offsets"), bias_classes_ptr=_at(s, "bias_classes"),
        bias_values_ptr=_at(s, "bias_values"), bias_count=s["bias_classes"].numel() if "bias_classes" in s else 0,
        allowed_ptr=_at(s, "allowed"), allowed_count=s["allowed"].shape[0] if "allowed" in s else 0,
        allowed_stride=s["allowed"].shape[1] if "allowed" in s else 0, allowed_rows_ptr=_at(s, "allowed_rows"))
    cb.adjust_scores(code, rows, classes, scores.data_ptr(), scores.stride(0), adjustment, result.data_ptr(), classes, stream)
    return result


def _own_top(s, cb, code, stream):
    case, scores = s["case"], s["scores"]
    rows, classes = scores.shape
    count, among = case["count"], case["among"]
    indexes = torch.empty(rows, count, dtype=torch.int32, device=DEVICE)
    weights = torch.empty(rows, count, dtype=torch.float64 if scores.dtype == torch.float64 else torch.float32, device=DEVICE)
    cb.select_top(code, rows, classes, scores.data_ptr(), scores.stride(0), count, among, indexes.data_ptr(), weights.data_ptr(), stream)
    out = [indexes, weights]
    if case["backward"]:
        dx = torch.empty(rows, classes, dtype=scores.dtype, device=DEVICE)
        cb.select_top_backward(code, rows, classes, scores.data_ptr(), scores.stride(0), count, among, indexes.data_ptr(),
                               weights.data_ptr(), s["gradients"].data_ptr(), dx.data_ptr(), classes, stream)
        out.append(dx)
    return out


def _own_dispatch(s, cb, code, stream):
    case, ids = s["case"], s["ids"]
    slots, width = ids.numel(), case["width"]
    places = torch.empty_like(ids)
    offsets = torch.empty(case["experts"] + 1, dtype=torch.int32, device=DEVICE)
    size = cb.sort_by_expert_bytes(slots, case["experts"])
    workspace = torch.empty(size, dtype=torch.uint8, device=DEVICE)
    cb.sort_by_expert(slots, case["experts"], ids.data_ptr(), places.data_ptr(), offsets.data_ptr(), workspace.data_ptr(), size, stream)
    cb.dispatch_rows(code, case["rows"], width, case["per_row"], s["source"].data_ptr(), width, places.data_ptr(),
                     s["sorted"].data_ptr(), slots, width, stream)
    return [places, offsets, s["sorted"]]


def _own_combine(s, cb, code, stream):
    case, rows = s["case"], s["sorted"]
    slots, width = rows.shape
    result = torch.empty(case["rows"], width, dtype=rows.dtype, device=DEVICE)
    cb.combine_rows(code, case["rows"], width, case["per_row"], rows.data_ptr(), slots, width, s["places"].data_ptr(), _at(s, "weights"),
                    result.data_ptr(), width, stream)
    out = [result]
    if case["backward"]:
        dw = torch.empty_like(s["weights"]) if case["weighted"] else None
        cb.combine_rows_backward(code, case["rows"], width, case["per_row"], s["gradients"].data_ptr(), width, rows.data_ptr(), slots, width,
                                 s["places"].data_ptr(), _at(s, "weights"), s["sorted_gradients"].data_ptr(), width,
                                 0 if dw is None else dw.data_ptr(), stream)
        out.append(s["sorted_gradients"])
        if dw is not None:
            out.append(dw)
    return out


def run(state):
    op = state["case"]["op"]
    if own:
        import catboost_amd as cb

        call = {"adjust": _own_adjust, "top": _own_top, "dispatch": _own_dispatch, "combine": _own_combine}[op]
        return call(state, cb, CODES[state["case"]["type"]], torch.cuda.current_stream().cuda_stream)
    return {"adjust": _plain_adjust, "top": _plain_top, "dispatch": _plain_dispatch, "combine": _plain_combine}[op](state)


# ---- what a pass cannot do without

def work(case):
    op, size = case["op"], SIZES[case["type"]]
    rows = case["rows"]
    if op == "adjust":
        n = rows * case["classes"]
        history, biases = rows * case["history"], rows * case["biases"]
        masks = min(case["masks"], rows) * ((case["classes"] + 31) // 32) * 4 + 4 * rows if case["masks"] else 0
        read = 4 * history + (24 * rows if history else 0) + 8 * biases + (8 * rows if biases else 0) + (4 * case["classes"] if case["class_bias"] else 0)
        return {"bytes": 2 * n * size + read + masks, "flops": n * (2 if case["class_bias"] else 1) + 5 * history + biases}
    if op == "top":
        n, acc = rows * case["classes"], 8 if case["type"] == "f64" else 4
        forward = n * size + rows * case["count"] * (4 + acc)
        if not case["backward"]:
            return {"bytes": forward, "flops": 4 * n}
        return {"bytes": forward + n * size + rows * case["count"] * acc, "flops": 8 * n}
    moved, kept = rows * case["width"], rows * case["per_row"] * (1 - case["dropped"]) * case["width"]
    slots = rows * case["per_row"]
    if op == "dispatch":
        return {"bytes": (moved + kept) * size + 8 * slots + 4 * case["experts"], "flops": slots}
    acc = 8 if case["type"] == "f64" else 4
    weights = slots * acc if case["weighted"] else 0
    forward = (moved + kept) * size + 4 * slots + weights
    if not case["backward"]:
        return {"bytes": forward, "flops": 2 * kept}
    return {"bytes": forward + (moved + kept) * size + weights, "flops": 5 * kept}


# ---- the definitions in 64 bits

def exact(case, seed):
    if case["rows"] * case.get("classes", 0) > 60_000_000:
        return None
    s = prepare(case, seed)
    return {"adjust": _exact_adjust, "top": _exact_top, "dispatch": _exact_dispatch, "combine": _exact_combine}[case["op"]](s, case)


def _exact_adjust(s, case):
    x = s["scores"].double().clone()
    rows, classes = x.shape
    size = rows * classes
    if "history" in s:
        lengths = s["history_offsets"][1:] - s["history_offsets"][:-1]
        row = torch.repeat_interleave(torch.arange(rows, device=DEVICE), lengths)
        within = torch.arange(row.numel(), device=DEVICE) - torch.repeat_interleave(s["history_offsets"][:-1], lengths)
        flat = row * classes + s["history"].long()
        behind = within >= s["prompts"].long()[row]
        shown, n = torch.unique(flat, return_counts=True)
        r = torch.div(shown, classes, rounding_mode="floor")
        v = x.view(-1)[shown] if x.is_contiguous() else x.reshape(-1)[shown]
        rep = s["repetition"].double()[r]
        v = torch.where(v > 0, v / rep, v * rep)
        x = x.reshape(-1)
        x[shown] = v
        made, n = torch.unique(flat[behind], return_counts=True)
        r = torch.div(made, classes, rounding_mode="floor")
        x[made] -= s["frequency"].double()[r] * n.double() + s["presence"].double()[r]
        x = x.view(rows, classes)
    if "class_bias" in s:
        x += s["class_bias"].double()[None, :]
    if "bias_classes" in s:
        lengths = s["bias_offsets"][1:] - s["bias_offsets"][:-1]
        row = torch.repeat_interleave(torch.arange(rows, device=DEVICE), lengths)
        flat = row * classes + s["bias_classes"].long()
        # a stable sort leaves a class's last entry at the end of its run
        ordered, at = torch.sort(flat, stable=True)
        end = torch.ones_like(ordered, dtype=torch.bool)
        end[:-1] = ordered[1:] != ordered[:-1]
        x = x.reshape(-1)
        x[ordered[end]] += s["bias_values"].double()[at[end]]
        x = x.view(rows, classes)
    if "allowed" in s:
        bit = torch.arange(32, device=DEVICE, dtype=torch.int32)
        table = ((s["allowed"][:, :, None] >> bit) & 1).bool().reshape(s["allowed"].shape[0], -1)[:, :classes]
        masked = s["allowed_rows"] >= 0
        x[masked] = x[masked].masked_fill(~table[s["allowed_rows"][masked].long()], float("-inf"))
    return x


def _exact_top(s, case):
    x = s["scores"].double()
    rows, classes = x.shape
    k = case["count"]
    none = x == float("-inf")
    # by rank: how many come before it
    order = torch.argsort(-x, dim=1, stable=True)[:, :k]
    taken = torch.gather(~none, 1, order)
    picked = torch.zeros_like(x, dtype=torch.bool).scatter_(1, order, taken)
    p = torch.softmax(torch.where(picked if case["among"] else ~none, x, float("-inf")), 1).nan_to_num(0.0)
    weights = torch.where(taken, torch.gather(p, 1, order), 0)
    out = [torch.where(taken, order, -1).to(torch.int32), weights]
    if case["backward"]:
        g = torch.zeros_like(x).scatter_(1, order, torch.where(taken, s["gradients"].double(), 0))
        out.append(p * (g - (g * p).sum(1, keepdim=True)))
    return out


def _exact_dispatch(s, case):
    experts, k = case["experts"], case["per_row"]
    flat = s["ids"].reshape(-1).long()
    counts = torch.bincount(flat[flat >= 0], minlength=experts)
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64, device=DEVICE), torch.cumsum(counts, 0)])
    slots = torch.nonzero(flat >= 0)[:, 0]
    order = slots[torch.argsort(flat[slots] * flat.numel() + slots)]
    places = torch.full_like(flat, -1)
    places[order] = torch.arange(order.numel(), device=DEVICE)
    rows = torch.zeros(flat.numel(), case["width"], dtype=torch.float64, device=DEVICE)
    rows[:order.numel()] = s["source"].double()[torch.div(order, k, rounding_mode="floor")]
    return [places.view(s["ids"].shape).to(torch.int32), offsets.to(torch.int32), rows]


def _exact_combine(s, case):
    y, k = s["sorted"].double(), case["per_row"]
    w = s["weights"].double() if case["weighted"] else torch.ones(case["rows"], k, dtype=torch.float64, device=DEVICE)
    out = torch.zeros(case["rows"], case["width"], dtype=torch.float64, device=DEVICE)
    dy, dw = torch.zeros_like(y) if case["backward"] else None, torch.zeros_like(w)
    for j in range(k):
        rows = torch.nonzero(s["places"][:, j] >= 0)[:, 0]
        at = s["places"][rows, j].long()
        out[rows] += w[rows, j, None] * y[at]
        if case["backward"]:
            g = s["gradients"].double()[rows]
            dy[at] = w[rows, j, None] * g
            dw[rows, j] = torch.sum(g * y[at], 1)
    return [out] + ([dy] if case["backward"] else []) + ([dw] if case["backward"] and case["weighted"] else [])
