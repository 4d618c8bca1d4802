"""Operators over rows of many classes (a vocabulary): a teacher's top logits, the loss of a student that is distilled
from them with its gradient, and the verification of tokens that such a student has drafted.

`listed()` and `draw()` give cases, `prepare()` makes their inputs, `run()` is one pass: the framework's entry points
where `own` is true, otherwise the same mathematics in elementary torch operations.  `exact()` is the definition in 64
bits.  Whole numbers are int32 tensors, in which -1 stands for the ABI's 0xffffffff ("none")."""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2}

# what the largest listed case moves, and holds; a drawn case stays below
MOST_BYTES = 2 * 2 * 4096 * 131072
MOST_HELD = 4 * 7 * 1024 * 131072
# share of the sequences, at least, of which a token is turned down (they read a row of either model, the others one row)
TURNED_DOWN = 0.5


def listed():
    return [
        # candidates for the next token of eight sequences being decoded
        {"name": "top_k_decode", "op": "top_k", "type": "f32", "classes": 32768, "stride": 0, "rows": 8, "k": 50,
         "temperature": 1.0, "norm": False, "masked": 0.0},
        # a teacher's pass over 2048 positions, of which 64 logits each and the row's norm are kept
        {"name": "top_k_teacher", "op": "top_k", "type": "bf16", "classes": 131072, "stride": 0, "rows": 2048, "k": 64,
         "temperature": 2.0, "norm": True, "masked": 0.0},
        # an odd vocabulary whose rows are padded, half of it masked (constrained answers), in half precision
        {"name": "top_k_masked", "op": "top_k", "type": "f16", "classes": 50257, "stride": 50304, "rows": 333, "k": 100,
         "temperature": 1.0, "norm": True, "masked": 0.5},
        # a classifier's head of 1000 classes, 256 samples: the smallest step, loss and gradient apart
        {"name": "distill_head", "op": "distill", "mode": "apart", "type": "f32", "classes": 1000, "stride": 0, "rows": 256,
         "k": 10, "temperature": 4.0, "norm": False},
        # the loss alone, on the few positions of a validation sample
        {"name": "distill_few", "op": "distill", "mode": "loss", "type": "bf16", "classes": 131072, "stride": 0, "rows": 24,
         "k": 64, "temperature": 1.0, "norm": True},
        # a training step's head, loss and gradient in one call, in 32 bits
        {"name": "distill_step_f32", "op": "distill", "mode": "step", "type": "f32", "classes": 32768, "stride": 0, "rows": 2048,
         "k": 32, "temperature": 2.0, "norm": False},
        # an odd vocabulary in half precision with padded rows, loss and gradient apart
        {"name": "distill_odd", "op": "distill", "mode": "apart", "type": "f16", "classes": 50257, "stride": 50304, "rows": 1001,
         "k": 33, "temperature": 1.5, "norm": True},
        # a training step of 4096 positions over a large vocabulary: the largest
        {"name": "distill_step", "op": "distill", "mode": "step", "type": "bf16", "classes": 131072, "stride": 0, "rows": 4096,
         "k": 64, "temperature": 1.0, "norm": True},
        # one sequence being decoded, four tokens drafted: nothing but latency
        {"name": "verify_one", "op": "verify", "classes": 131072, "drafted": 4, "sequences": 1, "point": False, "ragged": False},
        # a batch being served, drafts of different lengths
        {"name": "verify_batch", "op": "verify", "classes": 50257, "drafted": 5, "sequences": 64, "point": False, "ragged": True},
        # tokens drafted without a model (looked up in the prompt): the draft is a point mass
        {"name": "verify_lookup", "op": "verify", "classes": 32768, "drafted": 8, "sequences": 200, "point": True, "ragged": True},
        # the largest batch
        {"name": "verify_large", "op": "verify", "classes": 131072, "drafted": 3, "sequences": 1024, "point": False,
         "ragged": False},
    ]


def _spread(rng, lo, hi):
    """A whole number, spread evenly over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["top_k", "distill", "distill", "verify"])
    classes = _spread(rng, 1000, 131072)
    if rng.random() < 0.3:
        classes = max(1024, classes // 1024 * 1024)
    if op == "verify":
        drafted = rng.randint(1, 8)
        sequences = _spread(rng, 1, max(1, min(1024, MOST_HELD // (4 * (2 * drafted + 1) * classes))))
        return {"op": op, "classes": classes, "drafted": drafted, "sequences": sequences, "point": rng.random() < 0.3,
                "ragged": rng.random() < 0.5}
    kind = rng.choice(["f32", "bf16", "f16"])
    stride = 0 if rng.random() < 0.6 else (classes + 63) // 64 * 64
    passes = 1 if op == "top_k" else 3
    rows = _spread(rng, 1, max(1, min(4096, MOST_BYTES // (SIZES[kind] * passes * max(classes, stride)))))
    case = {"op": op, "type": kind, "classes": classes, "stride": stride, "rows": rows,
            "temperature": rng.choice([1.0, 1.0, 2.0, 4.0, 0.75]), "norm": rng.random() < 0.5}
    if op == "top_k":
        case.update(k=_spread(rng, 1, 512), masked=rng.choice([0.0, 0.0, 0.5, 0.99]))
    else:
        case.update(k=_spread(rng, 1, 256), mode=rng.choice(["loss", "apart", "step"]))
    return case


def _stride(case):
    return case["stride"] or case["classes"]


def _logits(case, gen):
    """Logits as a head gives them: a bell, and a tail of few likely classes; the padding holds anything."""
    rows, stride = case["rows"], _stride(case)
    out = torch.empty(rows, stride, dtype=TYPES[case["type"]], device="cuda")
    step = max(1, (1 << 27) // stride)
    for r in range(0, rows, step):
        z = torch.randn(min(step, rows - r), stride, generator=gen, device="cuda")
        out[r:r + step] = 1.5 * z + 0.1 * z * z.abs() + 0.02 * z * z * z
    return out


def _inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def uniform(*shape):
        return torch.rand(*shape, generator=gen, device="cuda")

    if case["op"] == "top_k":
        x = _logits(case, gen)
        if case["masked"]:
            step = max(1, (1 << 27) // x.shape[1])
            for r in range(0, x.shape[0], step):
                part = x[r:r + step]
                part.masked_fill_(uniform(*part.shape) < case["masked"], -math.inf)
        return {"x": x}
    if case["op"] == "distill":
        rows, classes, k, t = case["rows"], case["classes"], case["k"], case["temperature"]
        x = _logits(case, gen)
        # k different classes in an order of their own, their logits falling off; some rows hold fewer, a few none
        place = (torch.arange(k, device="cuda") + uniform(rows, k)) * (classes / k)
        index = place.long().clamp_(max=classes - 1).gather(1, uniform(rows, k).argsort(1))
        value = 9.0 - 1.2 * torch.log1p(torch.arange(k, device="cuda", dtype=torch.float32)) - uniform(rows, k)
        value = value.sort(1, descending=True)[0].to(TYPES[case["type"]]).float()
        # the student knows part of it
        near = (0.7 * value + 1.5 * torch.randn(rows, k, generator=gen, device="cuda")).to(x.dtype)
        x.scatter_(1, index, near)
        norm = None
        if case["norm"]:  # the slots hold between 80 and 99 hundredths of the teacher's mass
            norm = torch.logsumexp(value / t, 1) - torch.log(0.8 + 0.19 * uniform(rows))
        have = torch.where(uniform(rows) < 0.1, (uniform(rows) * (k + 1)).long(), k)
        absent = torch.arange(k, device="cuda") >= have[:, None]
        index = index.masked_fill(absent, -1).int()
        value = value.masked_fill(absent, -math.inf)
        # the mean over the positions; scaled by 2^16 where the gradient is in half precision, as its range asks for
        dy = (0.5 + uniform(rows)) / rows * (65536.0 if case["type"] == "f16" else 1.0)
        return {"x": x, "value": value, "index": index, "norm": norm, "dy": dy}
    classes, drafted, sequences = case["classes"], case["drafted"], case["sequences"]
    target = torch.empty(sequences, drafted + 1, classes, device="cuda")
    draft = None if case["point"] else torch.empty(sequences, drafted, classes, device="cuda")
    token = torch.empty(sequences, drafted, dtype=torch.int32, device="cuda")
    step = max(1, (1 << 26) // (classes * (drafted + 1)))
    for b in range(0, sequences, step):
        n = min(step, sequences - b)
        z = 2.5 * torch.randn(n, drafted + 1, classes, generator=gen, device="cuda")
        target[b:b + n] = torch.softmax(z, 2)
        z = z[:, :drafted]
        if draft is not None:
            z = z + 0.6 * torch.randn(z.shape, generator=gen, device="cuda")
        q = torch.softmax(z, 2)
        if draft is not None:
            draft[b:b + n] = q
            token[b:b + n] = torch.multinomial(q.reshape(-1, classes), 1, generator=gen).view(n, drafted).int()
        else:  # a likely token, whose probability is then raised: a text that repeats itself
            token[b:b + n] = q.argmax(2).int()
            for i in range(drafted):
                p = target[b:b + n, i]
                p *= 0.4
                p.scatter_add_(1, token[b:b + n, i:i + 1].long(), torch.full((n, 1), 0.6, device="cuda"))
    length = torch.full((sequences,), drafted, dtype=torch.int32, device="cuda")
    if case["ragged"]:
        length = (uniform(sequences) * (drafted + 1)).int().clamp_(max=drafted)
    return {"target": target, "draft": draft, "token": token, "length": length, "accept": uniform(sequences, drafted),
            "pick": uniform(sequences)}


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case

    def empty(*shape, dtype=torch.float32):
        return torch.empty(*shape, dtype=dtype, device="cuda")

    # the buffers that a program keeps for the results
    if case["op"] == "top_k":
        rows, k = case["rows"], case["k"]
        s["out"] = (empty(rows, k), empty(rows, k, dtype=torch.int32), empty(rows) if case["norm"] else None)
    elif case["op"] == "distill":
        rows = case["rows"]
        s["out"] = (empty(rows), empty(rows), empty(rows), None if case["mode"] == "loss" else torch.zeros_like(s["x"]))
    else:
        s["out"] = (empty(case["sequences"], case["drafted"] + 1, dtype=torch.int32), empty(case["sequences"], dtype=torch.int32))
    return s


def run(state):
    op = state["case"]["op"]
    if own:
        return {"top_k": _own_top_k, "distill": _own_distill, "verify": _own_verify}[op](state)
    return {"top_k": _plain_top_k, "distill": _plain_distill, "verify": _plain_verify}[op](state)


# ---- the framework's entry points ----


def _own_top_k(s):
    from anode_amd import gpu

    c = s["case"]
    value, index, norm = s["out"]
    gpu.call("anode_gpu_top_k_rows_" + c["type"], c["classes"], c["rows"], c["stride"], c["k"], c["temperature"], s["x"], value,
             index, norm)
    return [value, index] if norm is None else [value, index, norm]


def _own_distill(s):
    from anode_amd import gpu

    c = s["case"]
    loss, top, total, dx = s["out"]
    head = (c["classes"], c["rows"], c["stride"], c["k"], c["temperature"])
    teacher = (s["value"], s["index"], s["norm"])
    if c["mode"] == "step":
        gpu.call("anode_gpu_softmax_distill_fused_fwd_bwd_rows_" + c["type"], *head, s["x"], *teacher, s["dy"], loss, top, total, dx)
    else:
        gpu.call("anode_gpu_softmax_distill_rows_" + c["type"], *head, s["x"], *teacher, loss, top, total)
        if c["mode"] == "apart":
            gpu.call("anode_gpu_softmax_distill_bwd_rows_" + c["type"], *head, s["dy"], s["x"], *teacher, top, total, dx)
    return [loss, top, total] if dx is None else [loss, top, total, dx[:, :c["classes"]]]


def _own_verify(s):
    from anode_amd import gpu

    c = s["case"]
    token, accepted = s["out"]
    gpu.call("anode_gpu_verify_draft_packed_f32", c["classes"], c["drafted"], c["sequences"], s["target"], s["draft"], s["token"],
             s["length"], s["accept"], s["pick"], token, accepted)
    return [token, accepted]


# ---- plain forms ----


def _plain_top_k(s):
    c = s["case"]
    x = s["x"][:, :c["classes"]].float()
    value, index = torch.sort(x.masked_fill(x.isnan(), -math.inf), dim=1, descending=True, stable=True)
    value, index = value[:, :c["k"]], index[:, :c["k"]]
    index = index.masked_fill(value == -math.inf, -1).int()
    if c["k"] > c["classes"]:
        more = (c["rows"], c["k"] - c["classes"])
        value = torch.cat([value, value.new_full(more, -math.inf)], 1)
        index = torch.cat([index, index.new_full(more, -1)], 1)
    out = [value.contiguous(), index.contiguous()]
    if c["norm"]:
        top = x.amax(1, keepdim=True)
        base = torch.where(top == -math.inf, 0.0, top)  # a row of which the mask leaves nothing: -inf
        total = torch.exp((x - base) / c["temperature"]).sum(1)
        out.append(base[:, 0] / c["temperature"] + torch.log(total))
    return out


def _plain_distill(s):
    c = s["case"]
    t = c["temperature"]
    x = s["x"][:, :c["classes"]].float()
    top = x.amax(1, keepdim=True)
    e = torch.exp((x - top) / t)
    total = e.sum(1, keepdim=True)
    index, value = s["index"].long(), s["value"]
    there = (index >= 0) & (index < c["classes"]) & (value > -math.inf)
    some = there.any(1, keepdim=True)
    z = torch.where(there, value / t, -math.inf)
    if s["norm"] is None:
        z = z - torch.where(some, z.amax(1, keepdim=True), 0.0)
        norm = torch.log(torch.where(some, torch.exp(z).sum(1, keepdim=True), 1.0))
    else:
        norm = s["norm"][:, None]
    log_p = z - norm
    p = torch.exp(log_p)
    place = index.clamp(0, c["classes"] - 1)
    log_q = (x.gather(1, place) - top) / t - torch.log(total)
    loss = torch.where(p == 0, 0.0, p * (log_p - log_q)).sum(1)
    out = [loss, top[:, 0], total[:, 0]]
    if c["mode"] != "loss":
        grad = e * (p.sum(1, keepdim=True) / total)
        grad.scatter_add_(1, place, -p)
        grad *= s["dy"][:, None] / t
        out.append(torch.where(some, grad, 0.0).to(s["x"].dtype))
    return out


def _plain_verify(s):
    c = s["case"]
    classes, drafted = c["classes"], c["drafted"]
    target, draft, token = s["target"], s["draft"], s["token"].long()
    # in 64 bits: the product is exact there, and a sum's border is where the token changes
    p = target[:, :drafted].gather(2, token[:, :, None])[:, :, 0].double()
    q = 1.0 if draft is None else draft.gather(2, token[:, :, None])[:, :, 0].double()
    place = torch.arange(drafted, device=p.device)
    taken = (s["accept"].double() * q < p) & (place < s["length"][:, None])
    accepted = taken.int().cumprod(1).sum(1)
    row = torch.arange(c["sequences"], device=p.device)
    weight = target[row, accepted].double()
    there = (accepted < s["length"])[:, None]
    last = accepted.clamp(max=drafted - 1)
    if draft is None:
        rest = weight.scatter(1, token[row, last][:, None], 0.0)
    else:
        rest = (weight - draft[row, last].double()).clamp_(min=0.0)
    rest = torch.where(there, rest, weight)
    rest = torch.where((rest > 0).any(1, keepdim=True), rest, weight)
    upto = rest.cumsum(1)
    border = s["pick"].double()[:, None] * upto[:, -1:]
    drawn = (upto <= border).sum(1)
    end = torch.where(rest > 0, torch.arange(classes, device=p.device), 0).amax(1)
    drawn = torch.minimum(drawn, end)
    places = torch.arange(drafted + 1, device=p.device)
    out = torch.cat([token, token.new_full((c["sequences"], 1), -1)], 1)
    out = torch.where(places < accepted[:, None], out, -1)
    out = torch.where(places == accepted[:, None], drawn[:, None], out)
    return [out.int(), accepted.int()]


# ---- what a pass cannot do without ----


def work(case):
    if case["op"] == "verify":
        # the rows that the token is drawn from, and the few numbers of every drafted token
        rows = case["sequences"] * (1.0 if case["point"] else 1.0 + TURNED_DOWN)
        small = case["sequences"] * (24 * case["drafted"] + 16)
        return {"bytes": int(rows * case["classes"] * 4) + small, "flops": int(2 * rows * case["classes"])}
    n = case["rows"] * case["classes"]
    small = case["rows"] * (8 * case["k"] + 16)
    if case["op"] == "top_k":
        return {"bytes": n * SIZES[case["type"]] + small, "flops": n * (5 if case["norm"] else 1)}
    passes = {"loss": 1, "step": 2, "apart": 2}[case["mode"]]
    return {"bytes": passes * n * SIZES[case["type"]] + small, "flops": n * (4 if passes == 1 else 9)}


# ---- the definition in 64 bits ----


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "top_k":
        return _exact_top_k(case, s)
    return _exact_distill(case, s) if case["op"] == "distill" else _exact_verify(case, s)


def _exact_top_k(c, s):
    values, indexes, norms = [], [], []
    step = max(1, (1 << 25) // c["classes"])
    for r in range(0, c["rows"], step):
        x = s["x"][r:r + step, :c["classes"]].double()
        norms.append(torch.logsumexp(x / c["temperature"], 1))
        x = torch.cat([x, x.new_full((x.shape[0], c["k"]), -math.inf)], 1)
        order = torch.argsort(-x, dim=1, stable=True)[:, :c["k"]]
        v = x.gather(1, order)
        values.append(v)
        indexes.append(torch.where(v == -math.inf, -1, order).int())
    out = [torch.cat(values), torch.cat(indexes)]
    return out + [torch.cat(norms)] if c["norm"] else out


def _exact_distill(c, s):
    t, n = c["temperature"], c["classes"]
    outs = [[], [], [], []]
    step = max(1, (1 << 25) // n)
    for r in range(0, c["rows"], step):
        x = s["x"][r:r + step, :n].double() / t
        q = torch.softmax(x, 1)
        lq = torch.log_softmax(x, 1)
        index, value = s["index"][r:r + step].long(), s["value"][r:r + step].double()
        there = (index >= 0) & (index < n) & (value > -math.inf)
        p = torch.where(there, torch.exp(value / t - (0.0 if s["norm"] is None else s["norm"][r:r + step, None].double())), 0.0)
        if s["norm"] is None:
            p = p / torch.where(there.any(1, keepdim=True), p.sum(1, keepdim=True), 1.0)
        dense = torch.zeros_like(x).scatter_add_(1, torch.where(there, index, 0), p)
        taken = torch.where(there, index, 0)
        terms = torch.where(p > 0, p * (torch.log(torch.where(p > 0, p, 1.0)) - lq.gather(1, taken)), 0.0)
        outs[0].append(terms.sum(1))
        outs[1].append(x.amax(1) * t)
        outs[2].append(1.0 / q.amax(1))
        if c["mode"] != "loss":
            w = s["dy"][r:r + step, None].double() / t
            outs[3].append(w * (p.sum(1, keepdim=True) * q - dense))
    return [torch.cat(o) for o in outs if o]


def _exact_verify(c, s):
    tokens = torch.full((c["sequences"], c["drafted"] + 1), -1, dtype=torch.int32)
    accepted = torch.zeros(c["sequences"], dtype=torch.int32)
    drafts, lengths = s["token"].cpu(), s["length"].cpu()
    us, picks = s["accept"].cpu(), s["pick"].cpu()
    hit = s["target"][:, :c["drafted"]].gather(2, s["token"].long()[:, :, None]).cpu()
    if s["draft"] is not None:
        said = s["draft"].gather(2, s["token"].long()[:, :, None]).cpu()
    for b in range(c["sequences"]):
        n = 0
        while n < int(lengths[b]):
            q = 1.0 if s["draft"] is None else float(said[b, n])
            if not float(us[b, n]) * q < float(hit[b, n]):
                break
            tokens[b, n] = drafts[b, n]
            n += 1
        w = s["target"][b, n].double()
        if n < int(lengths[b]):
            left = w.clone()
            if s["draft"] is None:
                left[int(drafts[b, n])] = 0.0
            else:
                left = torch.relu(left - s["draft"][b, n].double())
            if bool((left > 0).any()):
                w = left
        upto = torch.cumsum(w, 0)
        over = upto > float(picks[b]) * upto[-1]
        first = torch.argmax(over.int()) if bool(over.any()) else torch.nonzero(w > 0)[-1, 0]
        tokens[b, n] = int(first)
        accepted[b] = n
    return [tokens, accepted]
