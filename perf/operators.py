"""The cases on which the document attention and the token embedding are measured.

Two operators with two passes each:

  attend    document attention, forward: causal attention inside every document of packed rows
            (validation passes, and the forward half of a training step);
  train     the same with its gradients: dq, dk, dv, the probabilities recomputed from q and k;
  lookup    token embedding: rows of the table, scaled, rounded to the compute dtype;
  gradient  the table's gradient: the output gradients of equal tokens summed, zero elsewhere.

`run` computes them in plain torch, or through the package where `own` is true.
"""

import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _attention(kind, name, rows, width, heads, kv_heads, head_dim, dtype, documents, low=1, high=None, gap=0, layout_seed=1):
    """documents "whole": every row is one document; "mixed": lengths log-uniform in [low, high], and after each
    document up to `gap` padding tokens."""
    return {"name": name, "kind": kind, "rows": rows, "width": width, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "dtype": dtype, "documents": documents, "low": low, "high": high or width, "gap": gap,
            "layout_seed": layout_seed}


def _embedding(kind, name, tokens, vocab, hidden, table, dtype, ids, scale=1.0, padding=-1):
    """ids "uniform", or "skewed": log-uniform, so that a few tokens make up most of the batch, as in text.
    `padding` >= 0 is the row that gets no gradient."""
    return {"name": name, "kind": kind, "tokens": tokens, "vocab": vocab, "hidden": hidden, "table": table, "dtype": dtype,
            "ids": ids, "scale": scale, "padding": padding}


def listed():
    return [
        # one short prompt through a 1.3B-class layer: latency
        _attention("attend", "attend_short_prompt", 1, 77, 16, 1, 128, "bf16", "whole"),
        # the 1.3B-class decoder's validation batch: 8 packed rows, documents of 64 to 4096 tokens
        _attention("attend", "attend_1b_packed", 8, 4096, 16, 1, 128, "bf16", "mixed", 64, 4096),
        # the 7B-class decoder on rows that are one document each
        _attention("attend", "attend_7b_whole_rows", 4, 4096, 32, 1, 128, "bf16", "whole"),
        # the tiny fp32 decoder: 2 packed rows of 512, documents of 32 to 256
        _attention("train", "train_tiny_fp32", 2, 512, 4, 1, 64, "fp32", "mixed", 32, 256),
        # the 7B-class decoder's training batch
        _attention("train", "train_7b_packed", 4, 4096, 32, 1, 128, "bf16", "mixed", 64, 4096),
        # short conversations with padding behind them, grouped heads, odd row length
        _attention("train", "train_grouped_ragged", 3, 2047, 24, 8, 64, "fp16", "mixed", 5, 600, gap=9),
        # one long document
        _attention("train", "train_long_document", 1, 16384, 16, 1, 128, "bf16", "whole"),
        # one short prompt's tokens
        _embedding("lookup", "lookup_short_prompt", 77, 49152, 4096, "bf16", "bf16", "uniform"),
        # the 7B-class batch out of the fp32 table that trains
        _embedding("lookup", "lookup_7b_trained", 16384, 49152, 4096, "fp32", "bf16", "uniform"),
        # the tiny decoder's table, scaled by the root of its width
        _embedding("gradient", "gradient_tiny", 1024, 1024, 256, "fp32", "fp32", "uniform", 16.0, 0),
        # the 7B-class batch
        _embedding("gradient", "gradient_7b_uniform", 16384, 49152, 4096, "fp32", "bf16", "uniform", 1.0, 0),
        # text: a few tokens make up most of the batch
        _embedding("gradient", "gradient_1b_text", 32768, 49152, 2048, "fp32", "bf16", "skewed", 1.0, 0),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(("attend", "train", "train", "lookup", "gradient"))
    if kind in ("attend", "train"):
        dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
        width = _log_int(rng, 1, 1024 if dtype == "fp32" else 11000)
        rows = rng.randint(1, max(1, min(6, 16384 // width)))
        kv_heads = rng.choice((1, 1, 2, 4))
        heads = kv_heads * rng.choice((1, 2, 3, 4, 8))
        head_dim = rng.choice((64, 128, 128, 32, 80, 96))
        documents = rng.choice(("whole", "mixed", "mixed"))
        high = _log_int(rng, 1, width)
        # many tiny documents only mean many small calls of the plain form: at most a few hundred of them
        low = max(rng.randint(1, high), min(high, rows * width // 300))
        return _attention(kind, "", rows, width, heads, kv_heads, head_dim, dtype, documents, low, max(high, low),
                          rng.choice((0, 0, 3, 40)), rng.randrange(1 << 30))
    tokens = _log_int(rng, 1, 20000)
    hidden = _log_int(rng, 32, 4096)
    vocab = _log_int(rng, 97, 49152)
    return _embedding(kind, "", tokens, vocab, hidden, rng.choice(("fp32", "bf16")) if kind == "lookup" else "fp32",
                      rng.choice(("bf16", "fp16", "fp32")), rng.choice(("uniform", "skewed")),
                      rng.choice((1.0, round(hidden ** 0.5, 3))), rng.choice((-1, 0)))


def _spans(case):
    """((row, start, end), ...): the documents, from the case alone."""
    if case["documents"] == "whole":
        return tuple((row, 0, case["width"]) for row in range(case["rows"]))
    rng, spans = random.Random(case["layout_seed"]), []
    for row in range(case["rows"]):
        start = 0
        while start < case["width"]:
            end = min(case["width"], start + _log_int(rng, case["low"], case["high"]))
            spans.append((row, start, end))
            start = end + (rng.randint(0, case["gap"]) if case["gap"] else 0)
    return tuple(spans)


def _make(case, seed):
    """The inputs of a case, from the seed."""
    generator = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda shape, dtype, factor=1.0: (torch.randn(shape, generator=generator, device="cuda") * factor).to(dtype)
    dtype = TYPES[case["dtype"]]
    if case["kind"] in ("attend", "train"):
        leading = (case["rows"], case["width"])
        q = normal((*leading, case["heads"], case["head_dim"]), dtype)
        k = normal((*leading, case["kv_heads"], case["head_dim"]), dtype)
        v = normal((*leading, case["kv_heads"], case["head_dim"]), dtype)
        return {"q": q, "k": k, "v": v, "dy": normal(q.shape, dtype) if case["kind"] == "train" else None}
    tokens, vocab = case["tokens"], case["vocab"]
    uniform = torch.rand(tokens, generator=generator, device="cuda", dtype=torch.float64)
    ids = uniform * vocab if case["ids"] == "uniform" else torch.exp(uniform * math.log(vocab)) - 1
    ids = ids.long().clamp_(0, vocab - 1)
    if case["kind"] == "lookup":
        return {"ids": ids, "weight": normal((vocab, case["hidden"]), TYPES[case["table"]], 0.02)}
    return {"ids": ids, "dy": normal((tokens, case["hidden"]), dtype)}


def prepare(case, seed):
    state = _make(case, seed)
    state["case"] = case
    if case["kind"] in ("attend", "train"):
        state["spans"] = _spans(case)
        if case["kind"] == "train":
            for name in ("q", "k", "v"):
                state[name].requires_grad_(True)
        if own:
            from causal_tuner_b200.kernels.attention_cuda import prepare_documents
            state["plan"] = prepare_documents(state["q"].shape[:2], state["spans"], state["q"].device, case["heads"],
                                              case["kv_heads"])
    return state


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    case = state["case"]
    if case["kind"] in ("attend", "train"):
        from causal_tuner_b200.kernels.attention_cuda import document_attention
        y = document_attention(state["q"], state["k"], state["v"], state["plan"])
        if case["kind"] == "attend":
            return {"y": y}
        dq, dk, dv = torch.autograd.grad(y, (state["q"], state["k"], state["v"]), state["dy"])
        return {"y": y.detach(), "dq": dq, "dk": dk, "dv": dv}
    from causal_tuner_b200.kernels.embedding_cuda import embedding_gradient, embedding_lookup
    if case["kind"] == "lookup":
        return {"x": embedding_lookup(state["ids"], state["weight"], scale=case["scale"], dtype=TYPES[case["dtype"]])}
    return {"d_weight": embedding_gradient(state["dy"], state["ids"], case["vocab"], scale=case["scale"],
                                           padding_idx=case["padding"] if case["padding"] >= 0 else None)}


@torch.no_grad()
def _run_plain(state):
    case = state["case"]
    if case["kind"] in ("attend", "train"):
        return _plain_attention(state, case["kind"] == "train")
    if case["kind"] == "lookup":
        return {"x": (state["weight"][state["ids"]].float() * case["scale"]).to(TYPES[case["dtype"]])}
    ids, dy = state["ids"], state["dy"].float()
    if case["padding"] >= 0:
        dy = dy * (ids != case["padding"]).unsqueeze(-1)
    total = torch.zeros((case["vocab"], case["hidden"]), device=dy.device, dtype=torch.float32)
    return {"d_weight": total.index_add_(0, ids, dy) * case["scale"]}


def _plain_attention(state, train):
    """Per document and group of heads: scores, causal mask, softmax, product; and the formulas of its gradient."""
    case = state["case"]
    q, k, v = (state[name].detach() for name in ("q", "k", "v"))
    group, scale = case["heads"] // case["kv_heads"], case["head_dim"] ** -0.5
    y = torch.zeros(q.shape, device=q.device, dtype=torch.float32)
    if train:
        dy = state["dy"]
        dq = torch.zeros(q.shape, device=q.device, dtype=torch.float32)
        dk = torch.zeros(k.shape, device=q.device, dtype=torch.float32)
        dv = torch.zeros(v.shape, device=q.device, dtype=torch.float32)
    for row, start, end in state["spans"]:
        length = end - start
        later = torch.ones((length, length), device=q.device, dtype=torch.bool).triu(1)
        step = max(1, min(group, (1 << 28) // (length * length)))
        for shared in range(case["kv_heads"]):
            keys, values = k[row, start:end, shared].float(), v[row, start:end, shared].float()
            for first in range(shared * group, (shared + 1) * group, step):
                heads = slice(first, min(first + step, (shared + 1) * group))
                queries = q[row, start:end, heads].float().transpose(0, 1)
                scores = (queries @ keys.T * scale).masked_fill_(later, float("-inf"))
                scores = torch.exp(scores - scores.amax(-1, keepdim=True))
                weights = scores / scores.sum(-1, keepdim=True)
                out = weights @ values
                y[row, start:end, heads] = out.transpose(0, 1)
                if train:
                    upstream = dy[row, start:end, heads].float().transpose(0, 1)
                    dv[row, start:end, shared] += (weights.transpose(1, 2) @ upstream).sum(0)
                    inner = (upstream * out).sum(-1, keepdim=True)
                    weights = weights * (upstream @ values.T - inner)
                    dq[row, start:end, heads] = (weights @ keys).transpose(0, 1) * scale
                    dk[row, start:end, shared] += (weights.transpose(1, 2) @ queries).sum(0) * scale
    result = {"y": y.to(q.dtype)}
    if train:
        result.update(dq=dq.to(q.dtype), dk=dk.to(q.dtype), dv=dv.to(q.dtype))
    return result


def exact(case, seed):
    inputs = _make(case, seed)
    if case["kind"] in ("attend", "train"):
        return _exact_attention(case, inputs)
    scale = case["scale"]
    if case["kind"] == "lookup":
        return {"x": torch.nn.functional.embedding(inputs["ids"], inputs["weight"].double()) * scale}
    # sorted tokens, running sums along them, differences at the ends of each token's run
    order = torch.argsort(inputs["ids"], stable=True)
    ids, result = inputs["ids"][order], torch.zeros((case["vocab"], case["hidden"]), device="cuda", dtype=torch.float64)
    present, counts = torch.unique_consecutive(ids, return_counts=True)
    ends = counts.cumsum(0).tolist()
    begin = 0
    for token, end in zip(present.tolist(), ends):
        if token != case["padding"]:
            result[token] = inputs["dy"][order[begin:end]].double().sum(0) * scale
        begin = end
    return {"d_weight": result}


def _exact_attention(case, inputs):
    """Block of queries by block of queries against all earlier keys, in 64 bits."""
    q, k, v, dy = (None if inputs[name] is None else inputs[name].double() for name in ("q", "k", "v", "dy"))
    group, scale = case["heads"] // case["kv_heads"], 1.0 / math.sqrt(case["head_dim"])
    results = [torch.zeros_like(t) for t in ((q,) if dy is None else (q, q, k, v))]
    for row, start, end in _spans(case):
        block = max(1, min(end - start, (1 << 26) // ((end - start) * group)))
        for first in range(start, end, block):
            last = min(end, first + block)
            hidden = torch.arange(start, last, device="cuda") > torch.arange(first, last, device="cuda").unsqueeze(1)
            for shared in range(case["kv_heads"]):
                mine = slice(shared * group, (shared + 1) * group)
                keys, values = k[row, start:last, shared], v[row, start:last, shared]
                scores = torch.einsum("qhd,kd->hqk", q[row, first:last, mine], keys) * scale
                weights = torch.softmax(scores.masked_fill(hidden, -math.inf), -1)
                results[0][row, first:last, mine] = torch.einsum("hqk,kd->qhd", weights, values)
                if dy is None:
                    continue
                upstream = dy[row, first:last, mine]
                results[3][row, start:last, shared] += torch.einsum("hqk,qhd->kd", weights, upstream)
                slope = torch.einsum("qhd,kd->hqk", upstream, values)
                slope = weights * (slope - (slope * weights).sum(-1, keepdim=True))
                results[1][row, first:last, mine] = torch.einsum("hqk,kd->qhd", slope, keys) * scale
                results[2][row, start:last, shared] += torch.einsum("hqk,qhd->kd", slope, q[row, first:last, mine]) * scale
    return dict(zip(("y", "dq", "dk", "dv"), results))


def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    if case["kind"] in ("attend", "train"):
        tokens = sum(end - start for _, start, end in _spans(case))
        pairs = sum((end - start) * (end - start + 1) // 2 for _, start, end in _spans(case))
        element = size[case["dtype"]] * case["head_dim"]
        whole = case["rows"] * case["width"] * case["heads"] * element      # outputs are written for padding too
        shared = case["rows"] * case["width"] * case["kv_heads"] * element
        read = tokens * (case["heads"] + 2 * case["kv_heads"]) * element
        if case["kind"] == "attend":
            return {"bytes": read + whole, "flops": 4 * pairs * case["heads"] * case["head_dim"]}
        return {"bytes": read + tokens * case["heads"] * element + 2 * whole + 2 * shared,
                "flops": 14 * pairs * case["heads"] * case["head_dim"]}
    entry, rows = size[case["dtype"]] * case["hidden"], case["tokens"]
    if case["kind"] == "lookup":
        # the rows that are asked for, each once: the expected number of different ids
        vocab, spread = case["vocab"], math.log(case["vocab"])
        share = [1 / vocab if case["ids"] == "uniform" else math.log1p(1 / (i + 1)) / spread for i in range(vocab)]
        distinct = sum(1 - (1 - p) ** rows for p in share)
        return {"bytes": int(rows * 8 + distinct * size[case["table"]] * case["hidden"] + rows * entry),
                "flops": rows * case["hidden"]}
    return {"bytes": rows * 8 + rows * entry + case["vocab"] * case["hidden"] * 4, "flops": rows * case["hidden"]}
