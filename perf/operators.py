"""Cases of the banded causal attention operators: what is measured, and their plain forms.

Two operators of the attention layers, forward and training (forward + backward):

* ``window``: causal attention in which a query sees the last ``window`` positions (its own
  included) and the first ``sinks`` keys of the sequence;
* ``bias``: causal attention whose scores get a learned bias ``table[head, bucket(distance)]``,
  optionally inside a window as well; its training form also returns the table's gradient.

Query row ``i`` stands at position ``query_start + i`` and key ``j`` at position ``j``; tensors are
``[batch, rows, heads, head_dim]`` in bf16.  ``heads_kv`` may divide ``heads`` (grouped heads).
"""
import math

import torch

own = False  # True: ``run`` calls the framework's kernels; False: the plain form below


def _case(name, op, train, batch, rows, keys, heads, heads_kv, dim, window=0, sinks=0, buckets=0, distance=0, layout="bshd"):
    # query rows are the last ones of the key sequence: a whole sequence when rows == keys, else a shard of it
    return {"name": name, "op": op, "train": train, "batch": batch, "rows": rows, "keys": keys, "heads": heads, "heads_kv": heads_kv,
            "dim": dim, "window": window, "sinks": sinks, "buckets": buckets, "distance": distance, "layout": layout}


def listed():
    return [
        # one short sequence, a handful of heads: an evaluation call, where launch latency is all
        _case("window fwd tiny", "window", False, 1, 60, 60, 4, 4, 64, 16, 0),
        # the 345M model's attention (2 x 2048 tokens, 16 heads of 64) with a narrow window, evaluation
        _case("window fwd 2x2048 d64", "window", False, 2, 2048, 2048, 16, 16, 64, 256, 4),
        # the same model in training with a window of a quarter of the sequence
        _case("window train 2x2048 d64", "window", True, 2, 2048, 2048, 16, 16, 64, 512, 4),
        # heads of 96 (760M model) straight from the packed projection, a length that ends inside a tile, a window that is no tile
        _case("window train 2x1999 d96", "window", True, 2, 1999, 1999, 16, 16, 96, 300, 1, layout="packed"),
        # heads of 128 (1.3B model) with grouped keys, long sequence, packed projection
        _case("window train 8192 gqa d128", "window", True, 1, 8192, 8192, 16, 2, 128, 1024, 16, layout="packed"),
        # a wide window over a long sequence, evaluation
        _case("window fwd 8192 d128", "window", False, 1, 8192, 8192, 16, 16, 128, 4096, 64),
        # one short odd sequence with a bias
        _case("bias fwd tiny", "bias", False, 1, 33, 33, 4, 4, 64, buckets=32, distance=128),
        # the 345M model's attention with a relative bias, training
        _case("bias train 2x2048 d64", "bias", True, 2, 2048, 2048, 16, 16, 64, buckets=32, distance=128),
        # ragged batch, grouped heads of 96, tensors laid out heads first, other bucket numbers, evaluation
        _case("bias fwd 3x777 gqa d96", "bias", False, 3, 777, 777, 12, 4, 96, buckets=20, distance=200, layout="bhsd"),
        # the 1.3B model's attention on a long sequence, training: the largest
        _case("bias train 8192 d128", "bias", True, 1, 8192, 8192, 16, 16, 128, buckets=32, distance=128),
        # the last rank's rows of a sequence split over four, bias inside a window with sinks, training
        _case("bias window train shard d128", "bias", True, 1, 2048, 8192, 16, 4, 128, 1024, 4, 32, 128),
        # the same mix on short sequences of a larger batch, training
        _case("bias window train 8x512 d64", "bias", True, 8, 512, 512, 16, 8, 64, 128, 2, 16, 64),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    op = rng.choice(("window", "bias"))
    train = rng.random() < 0.6
    dim = rng.choice((64, 96, 128))
    heads_kv = rng.choice((1, 2, 3, 4, 8, 16))
    heads = heads_kv * rng.choice([g for g in (1, 2, 3, 4, 8) if heads_kv * g <= 16])
    batch = rng.choice((1, 1, 2, 3, 4, 8))
    # a position that sees itself alone has a constant softmax: its training has nothing to compare, so two keys at least
    keys = _log_int(rng, 1 + train, 8192)
    while batch > 1 and batch * heads * keys * keys > 2 ** 29:
        batch -= 1
    rows = keys if rng.random() < 0.75 else _log_int(rng, 1, keys)
    window = _log_int(rng, 1 + train, 4096) if op == "window" or rng.random() < 0.4 else 0
    sinks = rng.choice((0, 1, 4, _log_int(rng, 1, 160))) if window else 0
    buckets = _log_int(rng, 2, 64) if op == "bias" else 0
    distance = buckets + _log_int(rng, 1, 256) if op == "bias" else 0
    layout = rng.choice(("bshd", "bhsd", "packed")) if rows == keys else rng.choice(("bshd", "bhsd"))
    case = _case("", op, train, batch, rows, keys, heads, heads_kv, dim, window, sinks, buckets, distance, layout)
    del case["name"]
    return case


def _tensors(case, seed, device):
    g = torch.Generator(device=device).manual_seed(seed)
    b, rows, keys, d = case["batch"], case["rows"], case["keys"], case["dim"]
    hq, hkv = case["heads"], case["heads_kv"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=device, dtype=torch.float32).to(torch.bfloat16)

    if case["layout"] == "packed":  # the three parts of one projection's output, in place
        q, k, v = normal(b, rows, (hq + 2 * hkv) * d).split([hq * d, hkv * d, hkv * d], dim=-1)
        q, k, v = q.unflatten(-1, (hq, d)), k.unflatten(-1, (hkv, d)), v.unflatten(-1, (hkv, d))
    elif case["layout"] == "bhsd":  # heads first in memory
        q, k, v = normal(b, hq, rows, d).transpose(1, 2), normal(b, hkv, keys, d).transpose(1, 2), normal(b, hkv, keys, d).transpose(1, 2)
    else:
        q, k, v = normal(b, rows, hq, d), normal(b, keys, hkv, d), normal(b, keys, hkv, d)
    dout = normal(b, rows, hq, d)
    table = normal(hq, case["buckets"]) if case["buckets"] else None
    return q, k, v, dout, table


def prepare(case, seed):
    q, k, v, dout, table = _tensors(case, seed, "cuda")
    leaves = [t.detach().requires_grad_(case["train"]) for t in (q, k, v) + (() if table is None else (table,))]
    return {"case": case, "leaves": leaves, "dout": dout, "scale": 1.0 / math.sqrt(case["dim"]),
            "limits": _limits(case["buckets"], case["distance"])}


def _limits(buckets, distance):
    """First distance of each bucket but bucket 0: the lower half of the buckets is one distance each, the rest is
    logarithmic up to ``distance``; whole numbers throughout, so that no distance falls on the wrong side of a border."""
    if not buckets:
        return None
    exact_ones = buckets // 2
    spread = buckets - exact_ones
    first, n = list(range(1, exact_ones + 1)), exact_ones
    for t in range(1, spread):
        while n ** spread * exact_ones ** t < distance ** t * exact_ones ** spread:
            n += 1
        first.append(n)
    return first


def run(state):
    case = state["case"]
    if own:
        from nano_megatron_b200.ops.band_attention import relative_bias_attention, window_attention

        start = case["keys"] - case["rows"]
        leaves = state["leaves"]
        if case["op"] == "window":
            out = window_attention(*leaves, state["scale"], window=case["window"], sinks=case["sinks"], query_start=start)
        else:
            out = relative_bias_attention(*leaves, state["scale"], max_distance=case["distance"], window=case["window"] or None,
                                          sinks=case["sinks"], query_start=start)
        if not case["train"]:
            return out
        return (out, *torch.autograd.grad(out, leaves, state["dout"]))
    with torch.no_grad():
        return _plain(state)


def _plain(state):
    case, scale = state["case"], state["scale"]
    q, k, v = (t.float() for t in state["leaves"][:3])
    b, rows, hq, d = q.shape
    keys, hkv = k.shape[1], k.shape[2]
    group = hq // hkv
    q = q.transpose(1, 2).reshape(b, hkv, group * rows, d)
    k, v = k.transpose(1, 2), v.transpose(1, 2)
    place = torch.arange(rows, device=q.device) + (keys - rows)
    key = torch.arange(keys, device=q.device)
    apart = place[:, None] - key[None, :]
    seen = apart >= 0
    if case["window"]:
        seen = seen & ((apart < case["window"]) | (key < case["sinks"])[None, :])
    scores = torch.matmul(q, k.transpose(-1, -2)).mul_(scale).view(b, hq, rows, keys)
    if case["op"] == "bias":
        limits = torch.tensor(state["limits"], device=q.device)
        bucket = torch.bucketize(apart.clamp(min=0), limits, right=True)
        scores += state["leaves"][3].float()[:, bucket]
    scores.masked_fill_(~seen, -math.inf)
    scores -= scores.amax(-1, keepdim=True)  # every row sees its own position
    probs = scores.exp_()
    probs /= probs.sum(-1, keepdim=True)
    probs = probs.view(b, hkv, group * rows, keys)
    out32 = torch.matmul(probs, v)
    out = out32.view(b, hq, rows, d).transpose(1, 2).to(torch.bfloat16)
    if not case["train"]:
        return out
    dout = state["dout"].float().transpose(1, 2).reshape(b, hkv, group * rows, d)
    dv = torch.matmul(probs.transpose(-1, -2), dout)
    dscores = torch.matmul(dout, v.transpose(-1, -2))
    dscores -= (dout * out32).sum(-1, keepdim=True)
    dscores *= probs
    dq = torch.matmul(dscores, k).mul_(scale).view(b, hq, rows, d).transpose(1, 2)
    dk = torch.matmul(dscores.transpose(-1, -2), q).mul_(scale).transpose(1, 2)
    grads = [t.to(torch.bfloat16) for t in (dq, dk, dv.transpose(1, 2))]
    if case["op"] == "bias":
        # sums along the diagonals of equal distance, then by bucket: row i of the reversed matrix starts one place further on
        across = keys + rows - 1
        slanted = torch.nn.functional.pad(dscores.view(b, hq, rows, keys).sum(0).flip(-1), (0, rows)).view(hq, -1)[:, :-rows]
        by_distance = slanted.reshape(hq, rows, across).sum(1, dtype=torch.float64)[:, rows - 1:]
        dtable = torch.zeros(hq, case["buckets"], device=q.device, dtype=torch.float64)
        dtable.index_add_(1, torch.bucketize(torch.arange(keys, device=q.device), limits, right=True), by_distance)
        grads.append(dtable.to(torch.bfloat16))
    return (out, *grads)


def _visible(case):
    """Pairs of a query and a key that it sees, for one head of one sequence."""
    start, window, sinks, keys = case["keys"] - case["rows"], case["window"], case["sinks"], case["keys"]
    if not window:
        return sum(p + 1 for p in range(start, keys))
    return sum(min(p + 1, window + min(sinks, max(0, p + 1 - window))) for p in range(start, keys))


def work(case):
    q = case["batch"] * case["rows"] * case["heads"] * case["dim"] * 2
    kv = case["batch"] * case["keys"] * case["heads_kv"] * case["dim"] * 2
    table = case["heads"] * case["buckets"] * 2
    pairs = case["batch"] * case["heads"] * _visible(case)
    if not case["train"]:
        return {"bytes": 2 * q + 2 * kv + table, "flops": 4 * case["dim"] * pairs}
    # q, k, v, dout in; out and the gradients out
    return {"bytes": 4 * q + 4 * kv + 2 * table, "flops": 14 * case["dim"] * pairs}


def exact(case, seed):
    q, k, v, dout, table = _tensors(case, seed, "cuda" if torch.cuda.is_available() else "cpu")
    rows, keys, group = case["rows"], case["keys"], case["heads"] // case["heads_kv"]
    start, scale = keys - rows, 1.0 / math.sqrt(case["dim"])
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    dq, dk, dv = torch.zeros_like(out), torch.zeros(k.shape, dtype=torch.float64, device=q.device), torch.zeros(k.shape, dtype=torch.float64, device=q.device)
    dtable = None if table is None else torch.zeros(table.shape, dtype=torch.float64, device=q.device)
    if table is not None:  # bucket of every distance, by counting up
        half, n_log = case["buckets"] // 2, case["buckets"] - case["buckets"] // 2
        of, b = [], 0
        for n in range(keys):
            if n < half:
                b = n
            else:
                b = max(b, half)
                while b + 1 < case["buckets"] and (n ** n_log) * half ** (b + 1 - half) >= case["distance"] ** (b + 1 - half) * half ** n_log:
                    b += 1
            of.append(b)
        of = torch.tensor(of, device=q.device)
    step = max(1, 2 ** 26 // keys)
    for b in range(case["batch"]):
        for h in range(case["heads"]):
            kh, vh = k[b, :, h // group].double(), v[b, :, h // group].double()
            for r0 in range(0, rows, step):
                r1 = min(rows, r0 + step)
                qh, g = q[b, r0:r1, h].double(), dout[b, r0:r1, h].double()
                away = torch.arange(start + r0, start + r1, device=q.device).unsqueeze(1) - torch.arange(keys, device=q.device)
                hidden = away < 0
                if case["window"]:
                    outside = away >= case["window"]
                    outside[:, : case["sinks"]] = False
                    hidden |= outside
                x = qh @ kh.t() * scale
                if table is not None:
                    at = of[away.clamp(min=0)]
                    x += table[h].double()[at]
                x[hidden] = -math.inf
                p = torch.exp(x - torch.logsumexp(x, 1, keepdim=True))
                out[b, r0:r1, h] = p @ vh
                if not case["train"]:
                    continue
                dv[b, :, h // group] += p.t() @ g
                dp = g @ vh.t()
                ds = p * (dp - (p * dp).sum(1, keepdim=True))
                dq[b, r0:r1, h] = ds @ kh * scale
                dk[b, :, h // group] += ds.t() @ qh * scale
                if table is not None:
                    for n in range(case["buckets"]):
                        dtable[h, n] += ds[at == n].sum()
    if not case["train"]:
        return out
    return (out, dq, dk, dv) if table is None else (out, dq, dk, dv, dtable)
