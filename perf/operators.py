"""Workloads of the operators around 8-bit scoring and beam selection.

Four operators of ``gustann_b200.api``:

``quantize_rows``   rows of float vectors to 8-bit codes and one scale a row
``matmul_i8``       products of 8-bit rows with both sides' scales and a bias
``beam_select``     the best k over beams and vocabulary
``reorder_states``  the states that follow the selected beams

Each case is a dict of plain values; ``run`` computes it in plain torch
operations, or with the framework's kernels when ``own`` is true.
"""
import math

import numpy as np
import torch

own = False

_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_DEV = "cuda"


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one text embedding, turned into codes before it is scored
        {"name": "quantize-one", "op": "quantize", "rows": 1, "dim": 768, "dtype": "f32"},
        # a slice of a base of text embeddings, turned into codes once
        {"name": "quantize-base", "op": "quantize", "rows": 500000, "dim": 768, "dtype": "f32"},
        # one query against a slice of the base: the smallest product, reads the codes once
        {"name": "score-one", "op": "matmul", "m": 1, "n": 100000, "k": 768, "out": "f32", "bias": False},
        # a few tokens against a vocabulary with an odd number of entries
        {"name": "score-vocab", "op": "matmul", "m": 24, "n": 32001, "k": 1024, "out": "bf16", "bias": True},
        # a linear layer of a text encoder over a ragged batch of tokens
        {"name": "linear-layer", "op": "matmul", "m": 4097, "n": 4096, "k": 4096, "out": "bf16", "bias": True},
        # a batch of queries against a slice of the base, squared distances through the bias
        {"name": "score-batch", "op": "matmul", "m": 4096, "n": 131072, "k": 768, "out": "f32", "bias": True},
        # one request's beams over a vocabulary
        {"name": "select-one", "op": "select", "groups": 1, "beams": 4, "vocab": 32001, "keep": 8, "dtype": "f32",
         "softmax": True, "finished": True},
        # a served batch of beams over a large vocabulary
        {"name": "select-batch", "op": "select", "groups": 64, "beams": 4, "vocab": 128000, "keep": 8,
         "dtype": "bf16", "softmax": True, "finished": True},
        # one level of codebook entries chosen by beam search for a block of vectors
        {"name": "select-codes", "op": "select", "groups": 100000, "beams": 8, "vocab": 256, "keep": 8, "dtype": "f32",
         "softmax": False, "finished": False},
        # the lists of eight parts joined into each query's best hundred
        {"name": "select-parts", "op": "select", "groups": 10000, "beams": 8, "vocab": 100, "keep": 100,
         "dtype": "f32", "softmax": False, "finished": False},
        # the codes chosen so far, behind one request's beams
        {"name": "reorder-one", "op": "reorder", "groups": 1, "beams": 4, "keep": 4, "heads": 1, "length": 33,
         "room": 64, "width": 1, "tensors": 1, "dtype": "f32"},
        # the caches of a served batch, a part of their room in use
        {"name": "reorder-batch", "op": "reorder", "groups": 16, "beams": 4, "keep": 4, "heads": 8, "length": 1023,
         "room": 1536, "width": 128, "tensors": 4, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["quantize", "matmul", "matmul", "select", "select", "select", "reorder"])
    if op == "quantize":
        dim = _log_int(rng, 1, 8192)
        rows = _log_int(rng, 1, max(1, min(1 << 19, 384000000 // dim)))
        return {"op": op, "rows": rows, "dim": dim, "dtype": rng.choice(sorted(_DT))}
    if op == "matmul":
        m = _log_int(rng, 1, 8192)
        n = _log_int(rng, 1, min(262144, 500000000 // m))
        k = _log_int(rng, 16, max(16, min(8192, 400000000000 // (m * n))))
        return {"op": op, "m": m, "n": n, "k": k, "out": rng.choice(sorted(_DT)), "bias": rng.random() < 0.5}
    if op == "select":
        kind = rng.choice(["tokens", "codes", "parts"])
        if kind == "tokens":
            beams = rng.randint(1, 16)
            vocab = _log_int(rng, 17, 200000)
            groups = _log_int(rng, 1, max(1, min(256, 32000000 // (beams * vocab))))
            keep = rng.randint(1, 2 * beams)
            dtype, softmax, fin = rng.choice(sorted(_DT)), True, rng.random() < 0.5
        elif kind == "codes":
            beams = _log_int(rng, 1, 32)
            vocab = _log_int(rng, 16, 4096)
            groups = _log_int(rng, 1, min(100000, 200000000 // (beams * vocab)))
            keep = _log_int(rng, 1, 32)
            dtype, softmax, fin = rng.choice(["f32", "f16"]), False, False
        else:
            beams = rng.randint(2, 64)
            vocab = _log_int(rng, 10, 128)
            groups = _log_int(rng, 1, 10000)
            keep = rng.randint(1, vocab)
            dtype, softmax, fin = "f32", False, False
        return {"op": op, "groups": groups, "beams": beams, "vocab": vocab, "keep": keep, "dtype": dtype,
                "softmax": softmax, "finished": fin}
    beams = rng.randint(1, 16)
    heads = rng.choice([1, 2, 8])
    width = rng.choice([1, 24, 64, 128, 129])
    tensors = rng.randint(1, 4)
    dtype = rng.choice(sorted(_DT))
    length = _log_int(rng, 1, 2048)
    per = beams * heads * width * tensors * length * 4
    groups = _log_int(rng, 1, max(1, min(64, 250000000 // per)))
    return {"op": op, "groups": groups, "beams": beams, "keep": rng.randint(1, beams), "heads": heads,
            "length": length, "room": length + rng.choice([0, 1, 64, length // 2]), "width": width,
            "tensors": tensors, "dtype": dtype}


# ------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device=_DEV)
    g.manual_seed(int(seed) * 2654435761 % (1 << 62) + 17)
    return g


def _vectors(rows, dim, g):
    """Embedding-like rows: normalised, a few dimensions larger than the rest."""
    x = torch.randn(rows, dim, generator=g, device=_DEV)
    gain = torch.ones(dim, device=_DEV)
    gain[torch.randint(0, dim, (max(1, dim // 100),), generator=g, device=_DEV)] = 6.0
    x *= gain
    x /= x.norm(dim=1, keepdim=True).clamp_min(1e-20)
    return x


def _padded(rows, dim, align):
    """An int8 matrix whose rows start on multiples of ``align`` bytes."""
    return torch.zeros(rows, (dim + align - 1) // align * align, dtype=torch.int8, device=_DEV)[:, :dim]


def _codes(rows, dim, g):
    """8-bit rows and scales as they follow from embedding-like vectors."""
    codes = _padded(rows, dim, 16)
    scales = torch.empty(rows, device=_DEV)
    step = max(1, (1 << 26) // dim)
    for s in range(0, rows, step):
        x = _vectors(min(step, rows - s), dim, g)
        a = x.abs().amax(1)
        scales[s:s + step] = a / 127
        codes[s:s + step] = torch.round(x * (127 / a)[:, None]).to(torch.int8)
    return codes, scales


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    if op == "quantize":
        x = _vectors(case["rows"], case["dim"], g)
        x[60::61] = 0  # padding rows
        return {"case": case, "x": x.to(_DT[case["dtype"]])}
    if op == "matmul":
        a, sa = _codes(case["m"], case["k"], g)
        b, sb = _codes(case["n"], case["k"], g)
        bias = torch.randn(case["n"], generator=g, device=_DEV) if case["bias"] else None
        return {"case": case, "a": a, "sa": sa, "b": b, "sb": sb, "bias": bias}
    if op == "select":
        n, w, v = case["groups"], case["beams"], case["vocab"]
        scores = -5.0 * torch.rand(n, w, generator=g, device=_DEV)
        logits = (3.0 * torch.randn(n, w, v, generator=g, device=_DEV)).to(_DT[case["dtype"]])
        finished = None
        if case["softmax"]:
            # tokens that may not follow
            hidden = torch.randint(0, v, (max(1, v // 50),), generator=g, device=_DEV)
            logits[:, :, hidden] = float("-inf")
            if n > 1:
                scores[0, 1:] = float("-inf")  # a request at its first token: one beam lives
        if case["finished"]:
            finished = torch.rand(n, w, generator=g, device=_DEV) < 0.2
        return {"case": case, "scores": scores, "logits": logits, "finished": finished, "end": v // 2}
    n, w, k = case["groups"], case["beams"], case["keep"]
    parents = torch.randint(0, w, (n, k), generator=g, device=_DEV, dtype=torch.int32)
    states = []
    for _ in range(case["tensors"]):
        t = torch.empty(n, w, case["heads"], case["room"], case["width"], dtype=_DT[case["dtype"]], device=_DEV)
        t.normal_(generator=g)
        states.append(t[:, :, :, :case["length"]])
    return {"case": case, "parents": parents, "states": states}


# ------------------------------------------------------------------- plain
def _plain_quantize(x):
    rows, dim = x.shape
    codes = torch.empty(rows, dim, dtype=torch.int8, device=x.device)
    scales = torch.empty(rows, dtype=torch.float32, device=x.device)
    step = max(1, (1 << 27) // dim)
    for s in range(0, rows, step):
        xs = x[s:s + step].float()
        sc = xs.abs().amax(1) / 127
        # the quotient decides which way a code rounds: 64 bits
        q = torch.round(xs.double() / sc.double()[:, None])
        codes[s:s + step] = torch.where(sc[:, None] > 0, q, torch.zeros_like(q)).to(torch.int8)
        scales[s:s + step] = sc
    return codes, scales


def _plain_matmul(a, sa, b, sb, bias, dtype):
    y = a.float() @ b.float().T
    y *= sa[:, None]
    y *= sb[None, :]
    if bias is not None:
        y += bias
    return y.to(dtype)


def _plain_select(scores, logits, keep, softmax, finished, end):
    n, w, v = logits.shape
    x = logits.double()
    x = torch.where(torch.isfinite(x), x, torch.full_like(x, float("-inf")))
    if softmax:
        top = x.amax(2, keepdim=True)
        top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
        x = (x - top) - (x - top).exp().sum(2, keepdim=True).log()
        x = torch.where(torch.isnan(x) | (x == float("inf")), torch.full_like(x, float("-inf")), x)
    if finished is not None:
        only = torch.full((v,), float("-inf"), dtype=torch.float64, device=x.device)
        only[end] = 0.0
        x = torch.where(finished[:, :, None], only, x)
    x = x + scores.double()[:, :, None]
    val, idx = torch.sort(x.reshape(n, w * v), dim=1, descending=True, stable=True)
    val, idx = val[:, :keep], idx[:, :keep]
    if val.shape[1] < keep:
        more = keep - val.shape[1]
        val = torch.cat([val, torch.full((n, more), float("-inf"), dtype=val.dtype, device=val.device)], 1)
        idx = torch.cat([idx, torch.zeros(n, more, dtype=idx.dtype, device=idx.device)], 1)
    ok = torch.isfinite(val)
    none = torch.full_like(idx, -1)
    return (val.float(), torch.where(ok, idx // v, none).int(), torch.where(ok, idx % v, none).int())


def _plain_reorder(states, parents):
    rows = torch.arange(parents.shape[0], device=parents.device)[:, None]
    return [s[rows, parents.long()] for s in states]


def run(state):
    c = state["case"]
    op = c["op"]
    if own:
        from gustann_b200 import api
        if op == "quantize":
            return api.quantize_rows(state["x"])
        if op == "matmul":
            return api.matmul_i8(state["a"], state["sa"], state["b"], state["sb"], bias=state["bias"],
                                 dtype=_DT[c["out"]])
        if op == "select":
            return api.beam_select(state["scores"], state["logits"], c["keep"], log_softmax=c["softmax"],
                                   finished=state["finished"], end_token=state["end"])
        return api.reorder_states(state["states"], state["parents"])
    if op == "quantize":
        return _plain_quantize(state["x"])
    if op == "matmul":
        return _plain_matmul(state["a"], state["sa"], state["b"], state["sb"], state["bias"], _DT[c["out"]])
    if op == "select":
        return _plain_select(state["scores"], state["logits"], c["keep"], c["softmax"], state["finished"],
                             state["end"])
    return _plain_reorder(state["states"], state["parents"])


# -------------------------------------------------------------- what it costs
def work(case):
    op = case["op"]
    if op == "quantize":
        n = case["rows"] * case["dim"]
        return {"bytes": n * (_DT[case["dtype"]].itemsize + 1) + 4 * case["rows"], "flops": 3 * n}
    if op == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": (m + n) * (k + 4) + m * n * _DT[case["out"]].itemsize + (4 * n if case["bias"] else 0),
                "flops": 2 * m * n * k}
    if op == "select":
        n = case["groups"] * case["beams"]
        out = 12 * case["groups"] * case["keep"]
        return {"bytes": n * case["vocab"] * _DT[case["dtype"]].itemsize + 5 * n + out,
                "flops": n * case["vocab"] * (4 if case["softmax"] else 1)}
    row = case["heads"] * case["length"] * case["width"] * case["tensors"] * _DT[case["dtype"]].itemsize
    # rows drawn at random: the distinct ones are read once, every kept one is written
    w, k = case["beams"], case["keep"]
    seen = w * (1 - (1 - 1 / w) ** k)
    return {"bytes": int(case["groups"] * row * (seen + k)) + 4 * case["groups"] * k, "flops": 0}


# -------------------------------------------------------------------- exact
def exact(case, seed):
    """The definitions in 64 bits, on the same inputs."""
    st = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        x = st["x"]
        codes, scales = [], []
        for part in torch.split(x, max(1, (1 << 26) // case["dim"])):
            p = part.double()
            top = torch.maximum(p.max(1).values, -p.min(1).values)
            step = (top / 127).float().double()           # codes are multiples of the stored, rounded scale
            q = p.abs() / torch.where(step > 0, step, torch.ones_like(step))[:, None]
            low = q.floor()
            up = (q - low > 0.5) | ((q - low == 0.5) & (low % 2 == 1))
            codes.append(((low + up) * p.sign()).to(torch.int8))
            scales.append(top / 127)
        return torch.cat(codes), torch.cat(scales)
    if op == "matmul":
        scaled = st["b"].double() * st["sb"].double()[:, None]
        out = []
        for a, sa in zip(torch.split(st["a"], 512), torch.split(st["sa"], 512)):
            y = torch.einsum("ik,jk->ij", a.double() * sa.double()[:, None], scaled)
            out.append(y if st["bias"] is None else y + st["bias"].double())
        return torch.cat(out)
    if op == "select":
        n, w, v, keep = case["groups"], case["beams"], case["vocab"], case["keep"]
        if n * w * v > 60000000 or n * w > 100000:
            if case["softmax"] or w * v < keep:
                return None
            val = [torch.topk((lg.double() + sc.double()[:, :, None]).flatten(1), keep, dim=1).values
                   for lg, sc in zip(torch.split(st["logits"], 4096), torch.split(st["scores"], 4096))]
            return torch.cat(val), None, None
        lg = st["logits"].float().cpu().numpy().astype(np.float64)
        sc = st["scores"].cpu().numpy().astype(np.float64)
        fin = st["finished"].cpu().numpy() if st["finished"] is not None else np.zeros((n, w), bool)
        val = np.full((n, keep), -np.inf)
        parent = np.full((n, keep), -1, np.int32)
        token = np.full((n, keep), -1, np.int32)
        for g in range(n):
            cand_v, cand_b, cand_t = [], [], []
            for b in range(w):
                row = lg[g, b]
                if not np.isfinite(sc[g, b]):
                    continue
                if fin[g, b]:
                    cand_v.append(sc[g, b:b + 1])
                    cand_b.append(np.array([b]))
                    cand_t.append(np.array([st["end"]]))
                    continue
                live = np.flatnonzero(np.isfinite(row))
                if live.size == 0:
                    continue
                x = row[live]
                if case["softmax"]:
                    m = x.max()
                    x = x - m - math.log(np.exp(x - m).sum())
                if live.size > keep:
                    edge = np.partition(x, live.size - keep)[live.size - keep]
                    near = x >= edge
                    x, live = x[near], live[near]
                cand_v.append(sc[g, b] + x)
                cand_b.append(np.full(live.size, b))
                cand_t.append(live)
            if not cand_v:
                continue
            cv, cb, ct = np.concatenate(cand_v), np.concatenate(cand_b), np.concatenate(cand_t)
            o = np.lexsort((ct, cb, -cv))[:keep]
            val[g, :o.size], parent[g, :o.size], token[g, :o.size] = cv[o], cb[o], ct[o]
        return (torch.from_numpy(val), torch.from_numpy(parent), torch.from_numpy(token))
    out = []
    for t in st["states"]:
        d = t.double()
        out.append(torch.stack([torch.stack([d[g, int(p)] for p in row])
                                for g, row in enumerate(st["parents"].tolist())]))
    return out
