"""The vocabulary operators: embedding lookup with scaling and its gradient by
sorted tokens, distillation from a teacher's top logits (loss, and loss with
gradient), and token sampling from given random numbers.

Each case names one call as a language model's training or serving loop makes
it. `run` computes it in plain torch operations, or through the package's own
entry points where `own` is true.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2}


# --- cases -------------------------------------------------------------------

def listed():
    return [
        # One decode step of a batch of sequences: a row per sequence.
        dict(name="lookup_decode", op="lookup", count=16, rows=131072, width=4096, dtype="bf16", ids="i32",
             scale=64.0, pad=0.0),
        # A packed training batch: every token of it, some of them padding.
        dict(name="lookup_batch", op="lookup", count=16384, rows=131072, width=4096, dtype="bf16", ids="i64",
             scale=64.0, pad=0.02),
        # A small model in full precision whose rows are no multiple of 16 bytes.
        dict(name="lookup_odd", op="lookup", count=5003, rows=50021, width=1021, dtype="f32", ids="i64",
             scale=1.0, pad=0.01),
        # The gradient of a short batch for a small table, in full precision.
        dict(name="gradient_small", op="gradient", count=2048, rows=32768, width=512, dtype="f32", out="f32",
             ids="i64", scale=1.0, pad=0.01, batches=1),
        # The gradient of a training batch: most of the table's rows get none.
        dict(name="gradient_batch", op="gradient", count=16384, rows=131072, width=2048, dtype="bf16", out="bf16",
             ids="i64", scale=45.25, pad=0.02, batches=1),
        # Two micro-batches into one gradient in full precision.
        dict(name="gradient_accumulate", op="gradient", count=20011, rows=32003, width=1544, dtype="f16", out="f32",
             ids="i32", scale=1.0, pad=0.02, batches=2),
        # The loss of an evaluation batch.
        dict(name="distill_eval", op="distill", grad=False, count=2048, rows=32768, stride=32768, top=64,
             dtype="bf16", teacher="f32", ids="i32", temperature=2.0, pad=0.02),
        # A training step on full-precision logits of a vocabulary of odd size.
        dict(name="distill_odd", op="distill", grad=True, count=509, rows=50021, stride=50021, top=33, dtype="f32",
             teacher="f32", ids="i64", temperature=1.0, pad=0.05),
        # A training step on a large vocabulary.
        dict(name="distill_train", op="distill", grad=True, count=4096, rows=131072, stride=131072, top=128,
             dtype="bf16", teacher="bf16", ids="i64", temperature=1.0, pad=0.02),
        # One sequence's next token.
        dict(name="sample_one", op="sample", count=1, rows=131072, stride=131072, dtype="f32", top_k=50, top_p=0.95,
             min_p=0.0, temperature=0.8, mixed=False),
        # A served batch with one setting for all: nucleus sampling alone.
        dict(name="sample_nucleus", op="sample", count=64, rows=131072, stride=131072, dtype="bf16", top_k=0,
             top_p=0.9, min_p=0.0, temperature=1.0, mixed=False),
        # A large served batch in which every request has settings of its own.
        dict(name="sample_mixed", op="sample", count=256, rows=100003, stride=100008, dtype="f32", top_k=0,
             top_p=1.0, min_p=0.0, temperature=1.0, mixed=True),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["lookup", "gradient", "gradient", "distill", "distill", "sample", "sample"])
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    ids = rng.choice(["i32", "i64"])
    rows = _log_int(rng, 1000, 131072)
    if op in ("lookup", "gradient"):
        count = _log_int(rng, 1 if op == "lookup" else 64, 16384)
        width = _log_int(rng, 64, 4096)
        if rng.random() < 0.7:  # most models' rows are a multiple of 64
            width = max(64, width // 64 * 64)
        pad = rng.choice([0.0, 0.01, 0.3])
        scale = rng.choice([1.0, width ** 0.5])
        if op == "lookup":
            return dict(op=op, count=count, rows=rows, width=width, dtype=dtype, ids=ids, scale=scale, pad=pad)
        width = min(width, 2048)
        return dict(op=op, count=count, rows=rows, width=width, dtype=dtype, out=rng.choice([dtype, "f32"]), ids=ids,
                    scale=scale, pad=pad, batches=rng.choice([1, 1, 2]))
    stride = rows if rng.random() < 0.6 else (rows + 127) // 64 * 64
    if op == "distill":
        count = min(_log_int(rng, 1, 4096), (1 << 28) // rows)
        return dict(op=op, grad=rng.random() < 0.7, count=count, rows=rows, stride=stride, top=_log_int(rng, 1, 256),
                    dtype=dtype, teacher=rng.choice(["f32", "bf16"]), ids=ids,
                    temperature=rng.choice([0.5, 1.0, 2.0, 4.0]), pad=rng.choice([0.0, 0.02, 0.3]))
    count = _log_int(rng, 1, 256)
    return dict(op=op, count=count, rows=rows, stride=stride, dtype=dtype,
                top_k=rng.choice([0, 0, 1, _log_int(rng, 2, 2000)]), top_p=rng.choice([1.0, 0.95, 0.8, 0.3]),
                min_p=rng.choice([0.0, 0.0, 0.02, 0.1]), temperature=rng.choice([0.0, 0.6, 1.0, 1.5]),
                mixed=rng.random() < 0.4)


# --- inputs ------------------------------------------------------------------

def _tokens(count, rows, ids, pad, gen):
    """Token numbers that fall off as one over their rank; -1 marks padding,
    at the end of the batch as a padded batch has it."""
    u = torch.rand(count, device="cuda", generator=gen, dtype=torch.float64)
    tokens = (torch.exp(u * math.log(rows + 1)) - 1).long().clamp_(0, rows - 1)
    used = count - int(count * pad)
    tokens[used:] = -1
    return tokens.int() if ids == "i32" else tokens


def _padded(x, stride):
    """The same matrix with `stride` elements from row to row."""
    if stride == x.shape[1]:
        return x
    base = torch.zeros(x.shape[0], stride, dtype=x.dtype, device=x.device)
    base[:, :x.shape[1]] = x
    return base[:, :x.shape[1]]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    def rand(*shape):
        return torch.rand(*shape, device="cuda", generator=gen)

    state = dict(case=case)
    count, rows = case["count"], case["rows"]
    if case["op"] == "lookup":
        state["table"] = (randn(rows, case["width"]) * 0.02).to(DTYPES[case["dtype"]])
        state["tokens"] = _tokens(count, rows, case["ids"], case["pad"], gen)
    elif case["op"] == "gradient":
        state["grads"] = [randn(count, case["width"]).to(DTYPES[case["dtype"]]) for _ in range(case["batches"])]
        state["tokens"] = [_tokens(count, rows, case["ids"], case["pad"], gen) for _ in range(case["batches"])]
        state["out"] = torch.zeros(rows, case["width"], dtype=DTYPES[case["out"]], device="cuda")
    elif case["op"] == "distill":
        top = min(case["top"], rows)
        # One token from each of `top` equal ranges, so that none is twice there.
        at = (torch.arange(top, device="cuda") + rand(count, top)) * (rows / top)
        at = torch.minimum(at.long(), torch.arange(1, top + 1, device="cuda") * rows // top - 1).clamp_(min=0)
        at = torch.maximum(at, -((-torch.arange(top, device="cuda") * rows) // top))
        at = at.gather(1, rand(count, top).argsort(1))
        teacher = (randn(count, top) * 3 + 8).sort(1, descending=True).values
        logits = randn(count, rows) * 2.5
        logits.scatter_add_(1, at, teacher * 0.6)
        cut = count - int(count * case["pad"])
        at[cut:] = -1  # padded positions have no teacher
        at[::7, (top + 1) // 2:] = -1  # and some have fewer top logits
        state["logits"] = _padded(logits.to(DTYPES[case["dtype"]]), case["stride"])
        state["at"] = at.int() if case["ids"] == "i32" else at
        state["teacher"] = teacher.to(DTYPES[case["teacher"]])
        state["weights"] = (rand(count) + 0.5) / count
    else:
        logits = randn(count, rows) * 2.5
        # Between flat and sharp rows: a dozen tokens stand out by 0 to 18.
        strong = (rand(count, 12) * rows).long()
        logits.scatter_add_(1, strong, rand(count, 1) * 14 + rand(count, 12) * 4)
        state["logits"] = _padded(logits.to(DTYPES[case["dtype"]]), case["stride"])
        state["uniform"] = rand(count)
        if case["mixed"]:
            pick = torch.arange(count, device="cuda")
            some = (rand(count) < 0.5)
            state["temperature"] = torch.where(pick % 8 == 0, 0.0, 0.5 + rand(count))
            state["top_k"] = torch.where(some, (rand(count) * 200).int() + 1, 0).int()
            state["top_p"] = torch.where(pick % 3 == 0, 1.0, 0.3 + 0.7 * rand(count))
            state["min_p"] = torch.where(pick % 5 == 0, 0.1 * rand(count), 0.0)
        else:
            for key in ("temperature", "top_k", "top_p", "min_p"):
                state[key] = case[key]
    return state


# --- the operators in plain form -----------------------------------------------

def _plain_lookup(state):
    table, tokens, case = state["table"], state["tokens"].long(), state["case"]
    found = (tokens >= 0) & (tokens < table.shape[0])
    picked = table[tokens.clamp(0, table.shape[0] - 1)].float() * case["scale"]
    return torch.where(found[:, None], picked, 0.0).to(table.dtype)


def _plain_gradient(state):
    case = state["case"]
    tokens = torch.cat(state["tokens"]).long()
    grads = torch.cat(state["grads"]).float()
    total = torch.zeros(case["rows"] + 1, case["width"], device="cuda")
    # Tokens outside of the table fall into a row behind it.
    tokens = torch.where((tokens >= 0) & (tokens < case["rows"]), tokens, case["rows"])
    total.index_add_(0, tokens, grads)
    return (total[:case["rows"]] * case["scale"]).to(state["out"].dtype)


def _plain_distill(state):
    case, t = state["case"], state["case"]["temperature"]
    z = state["logits"].float() / t
    peak = z.amax(1, keepdim=True)
    e = torch.exp(z - peak)
    mass = e.sum(1, keepdim=True)
    at = state["at"].long()
    used = (at >= 0) & (at < case["rows"])
    s = torch.where(used, state["teacher"].float() / t, -math.inf)
    s = s - s.amax(1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(s)
    total = p.sum(1, keepdim=True)
    some = total > 0
    p = torch.where(some, p / total.clamp(min=1e-30), 0.0)
    log_p = s - torch.log(total.clamp(min=1e-30))
    log_q = z.gather(1, at.clamp(0, case["rows"] - 1)) - peak - torch.log(mass)
    loss = t * t * torch.where(used, p * (log_p - log_q), 0.0).sum(1)
    if not case["grad"]:
        return loss
    weight = torch.where(some, state["weights"][:, None] * t, 0.0)
    g = e * (weight / mass)
    g.scatter_add_(1, at.clamp(0, case["rows"] - 1), torch.where(used, -weight * p, 0.0))
    return loss, g.to(state["logits"].dtype)


def _column(value, count, dtype):
    """A setting of one number, or of one for each row, as a column; numbers
    are rounded to 32 bits as the settings of a row are."""
    if not isinstance(value, torch.Tensor):
        value = torch.full((count,), value, dtype=torch.int32 if dtype == torch.int64 else torch.float32,
                           device="cuda")
    return value.to(dtype)[:, None]


def _plain_sample(state):
    x = state["logits"].double()
    count, rows = x.shape
    temperature = _column(state["temperature"], count, torch.float64)
    top_k = _column(state["top_k"], count, torch.int64)
    top_p = _column(state["top_p"], count, torch.float64)
    min_p = _column(state["min_p"], count, torch.float64)
    peak = x.amax(1, keepdim=True)
    w = torch.exp((x - peak) / torch.where(temperature > 0, temperature, 1.0))
    # The greatest first, of equal ones the lowest index.
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    w = w.gather(1, order)
    rank = torch.arange(rows, device="cuda")[None, :]
    kept = (top_k <= 0) | (rank < top_k)
    kept = kept & ((temperature > 0) | (rank < 1))
    w = torch.where(kept, w, 0.0)
    before = torch.cumsum(w, 1) - w
    kept = kept & ((top_p >= 1) | (before < top_p * w.sum(1, keepdim=True)) | (rank < 1)) & (w >= min_p)
    w = torch.where(kept, w, 0.0)
    back = torch.zeros_like(w).scatter_(1, order, w)
    sums = torch.cumsum(back, 1)
    over = (back > 0) & (sums > state["uniform"].double()[:, None] * sums[:, -1:])
    return over.int().argmax(1).int()


def run(state):
    case = state["case"]
    if own:
        import moderngpu_b200 as mgpu
        if case["op"] == "lookup":
            return mgpu.embedding_lookup(state["table"], state["tokens"], scale=case["scale"])
        if case["op"] == "gradient":
            for i in range(case["batches"]):
                mgpu.embedding_gradient(state["grads"][i], state["tokens"][i], case["rows"], scale=case["scale"],
                                        out=state["out"], accumulate=i > 0)
            return state["out"]
        if case["op"] == "distill":
            if not case["grad"]:
                return mgpu.distill_loss(state["logits"], state["at"], state["teacher"],
                                         temperature=case["temperature"])
            return mgpu.distill_loss_gradient(state["logits"], state["at"], state["teacher"],
                                              row_weights=state["weights"], temperature=case["temperature"])
        return mgpu.sample_tokens(state["logits"], state["uniform"], temperature=state["temperature"],
                                  top_k=state["top_k"], top_p=state["top_p"], min_p=state["min_p"])
    if case["op"] == "lookup":
        return _plain_lookup(state)
    if case["op"] == "gradient":
        return _plain_gradient(state)
    if case["op"] == "distill":
        return _plain_distill(state)
    return _plain_sample(state)


# --- what a pass cannot do without -----------------------------------------------

def _distinct(count, rows):
    """How many different tokens `count` draws of _tokens have on average."""
    v = np.arange(rows, dtype=np.float64)
    p = np.log((v + 2) / (v + 1)) / math.log(rows + 1)
    return float(np.sum(-np.expm1(count * np.log1p(-p))))


def work(case):
    count, rows = case["count"], case["rows"]
    if case["op"] in ("lookup", "gradient"):
        width, size = case["width"], SIZES[case["dtype"]]
        id_size = 4 if case["ids"] == "i32" else 8
        used = count - int(count * case["pad"])
        if case["op"] == "lookup":
            read = _distinct(used, rows) * width * size
            return {"bytes": read + count * (width * size + id_size), "flops": used * width}
        # The first micro-batch writes every row of the result, a later one
        # reads and writes those of its tokens.
        again = 2 * _distinct(used, rows) * (case["batches"] - 1)
        return {"bytes": case["batches"] * (used * width * size + count * id_size)
                + (rows + again) * width * SIZES[case["out"]],
                "flops": case["batches"] * used * width + rows * width}
    size = SIZES[case["dtype"]]
    if case["op"] == "distill":
        top = min(case["top"], rows)
        small = count * (top * (SIZES[case["teacher"]] + (4 if case["ids"] == "i32" else 8)) + 4)
        if not case["grad"]:
            return {"bytes": count * rows * size + small, "flops": 4 * count * rows}
        return {"bytes": 2 * count * rows * size + small + 4 * count, "flops": 6 * count * rows}
    return {"bytes": count * (rows * size + 8), "flops": 4 * count * rows}


# --- the definitions in 64 bits ---------------------------------------------------

def _exact_sample_row(x, u, temperature, top_k, top_p, min_p):
    if temperature <= 0:
        return int(np.argmax(x))
    order = np.argsort(-x, kind="stable")
    if top_k > 0:
        order = order[:top_k]
    w = np.exp((x[order] - x[order[0]]) / temperature)
    if top_p < 1:
        sums = np.cumsum(w)
        enough = int(np.searchsorted(sums, top_p * sums[-1], side="left")) + 1
        order, w = order[:enough], w[:enough]
    order = order[w >= min_p]
    order.sort()
    sums = np.cumsum(np.exp((x[order] - x.max()) / temperature))
    return int(order[min(np.searchsorted(sums, u * sums[-1], side="right"), len(order) - 1)])


def exact(case, seed):
    state = prepare(case, seed)
    count, rows = case["count"], case["rows"]
    if case["op"] == "lookup":
        tokens = state["tokens"].long()
        out = torch.zeros(count, case["width"], dtype=torch.float64, device="cuda")
        live = torch.nonzero((tokens >= 0) & (tokens < rows)).flatten()
        out[live] = torch.index_select(state["table"], 0, tokens[live]).double() * case["scale"]
        return out
    if case["op"] == "gradient":
        out = torch.zeros(rows, case["width"], dtype=torch.float64, device="cuda")
        for grad, tokens in zip(state["grads"], state["tokens"]):
            tokens = tokens.long()
            live = torch.nonzero((tokens >= 0) & (tokens < rows)).flatten()
            out.index_put_((tokens[live],), grad[live].double() * case["scale"], accumulate=True)
        return out
    if case["op"] == "distill":
        t = float(case["temperature"])
        loss = torch.zeros(count, dtype=torch.float64, device="cuda")
        grad = torch.zeros(count, rows, dtype=torch.float64, device="cuda") if case["grad"] else None
        step = max(1, (1 << 25) // rows)
        for a in range(0, count, step):
            b = min(count, a + step)
            log_q = torch.log_softmax(state["logits"][a:b].double() / t, dim=1)
            at = state["at"][a:b].long()
            p = torch.zeros_like(log_q)
            live = at >= 0
            at = at.clamp(min=0)
            top = torch.where(live, state["teacher"][a:b].double() / t, -math.inf)
            top = torch.nan_to_num(torch.softmax(top, dim=1), nan=0.0)
            p.scatter_add_(1, at, top)
            entropy = torch.special.entr(top).sum(1)
            loss[a:b] = t * t * (-entropy - (p * log_q).sum(1))
            if grad is not None:
                has = live.any(1).double()[:, None]
                grad[a:b] = state["weights"][a:b].double()[:, None] * t * (torch.exp(log_q) * has - p)
        return loss if grad is None else (loss, grad)
    host = {key: (state[key].cpu().numpy() if isinstance(state[key], torch.Tensor)
                  else np.full(count, state[key], np.int32 if key == "top_k" else np.float32))
            for key in ("temperature", "top_k", "top_p", "min_p", "uniform")}
    x = state["logits"].double().cpu().numpy()
    picked = [_exact_sample_row(x[i], float(host["uniform"][i]), float(host["temperature"][i]),
                                int(host["top_k"][i]), float(host["top_p"][i]), float(host["min_p"][i]))
              for i in range(count)]
    return torch.tensor(picked, dtype=torch.int32, device="cuda")
