"""What generating several answers to one prompt asks of the engine, as cases that can be timed and compared.

Two operators belong together there. The requests that answer one prompt hold the same pages for it, so their single tokens'
attention reads those pages once for all of them (`shared_prefix_attention`); and what makes the answers differ is the draw of
each next token under a request's own temperature, top_k, top_p and min_p (`sample_filtered`).

The fields of an "attention" case, one decoding step (every request brings one token):
  dtype                 "bfloat16" (serving) or "float32" (the true 32-bit path)
  heads, kv_heads, dim  query heads over key/value heads of this size (`v_dim`: the values' size where it is another)
  groups                requests that share a prompt, group after group, as text ("24,7")
  prefix                positions that each group shares, whole pages ("2048,640")
  alone                 further requests that share nothing; each holds up to `own` positions
  own                   the most positions a request holds of its own behind what it shares, its newest included
  window                0, or a row sees only its last `window` positions
  softcap               0, or scores are softcap * tanh(score / softcap)
  sinks                 whether a learned sink a head joins the denominator

The fields of a "sampling" case:
  rows, vocab           logits [rows, vocab] in float32
  filters               which settings the requests have: "top_k", "top_p", "min_p", "top_k top_p" (what a chat's defaults set), "mixed"
                        (requests of every kind in one step, plain and greedy ones among them)
  spread                how peaked the logits are: their standard deviation before a few hundred likely tokens are lifted above the rest
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

PAGE = 16                # positions a page of the engine's cache holds


# ---------------------------------------------------------------------------------------- the cases
def _attention(name, heads, kv_heads, dim, groups, prefix, own_tokens, dtype="bfloat16", alone=0, window=0, softcap=0.0, sinks=False, v_dim=0):
    return {"name": name, "kind": "attention", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "dim": dim, "v_dim": v_dim or dim,
            "groups": groups, "prefix": prefix, "alone": alone, "own": own_tokens, "window": window, "softcap": softcap, "sinks": sinks}


def _sampling(name, rows, vocab, filters, spread):
    return {"name": name, "kind": "sampling", "rows": rows, "vocab": vocab, "filters": filters, "spread": spread}


def listed():
    return [
        # Two answers to a chat's short prompt on Gemma 2 2B: latency and launches count.
        _attention("2 answers short", 8, 4, 256, "2", "192", 40, softcap=50.0),
        # Eight answers to the benchmark's 6,144 tokens on Gemma 2 2B.
        _attention("8 answers 6144", 8, 4, 256, "8", "6144", 300, softcap=50.0),
        # A batch of 64 answers on Gemma 2 9B, for best-of-n or a reward model.
        _attention("64 answers 2048", 16, 8, 256, "64", "2048", 500, softcap=50.0),
        # Requests of two system prompts beside requests of their own, on Gemma 2 27B's windowed layers: the longer prompt passes the window.
        _attention("two prompts windowed", 32, 16, 128, "24,7", "5008,640", 700, alone=3, window=4096, softcap=50.0),
        # A layer without a soft cap and with a sink a head, 16 heads over 4 of 128, a few odd lengths.
        _attention("19 answers sinks", 16, 4, 128, "19", "1008", 77, sinks=True),
        # The 32-bit path, which results are checked against.
        _attention("8 answers float32", 8, 4, 256, "8", "1024", 100, dtype="float32", softcap=50.0),
        # The largest: 128 answers to a long document on Gemma 2 27B's heads.
        _attention("128 answers 16384", 32, 16, 128, "128", "16384", 512, softcap=50.0),
        # One user's chat with the usual defaults, over Gemma 2's vocabulary.
        _sampling("1 row top_k top_p", 1, 256000, "top_k top_p", 2.0),
        # A small server's batch, each request with settings of its own.
        _sampling("8 rows mixed", 8, 256000, "mixed", 2.5),
        # A batch of answers drawn from the nucleus alone: no bound on how many tokens it keeps.
        _sampling("64 rows top_p", 64, 256000, "top_p", 1.5),
        # A smaller vocabulary of odd size, a floor relative to the likeliest token.
        _sampling("24 rows min_p odd", 24, 50257, "min_p", 3.0),
        # The largest batch that the engine records.
        _sampling("256 rows mixed", 256, 256000, "mixed", 2.0),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.4:
        vocab = rng.choice([256000, 256000, _log_uniform(rng, 300, 256000)])
        return {"kind": "sampling", "rows": _log_uniform(rng, 1, 256), "vocab": vocab,
                "filters": rng.choice(["top_k", "top_p", "min_p", "top_k top_p", "mixed"]), "spread": rng.choice([1.0, 1.5, 2.0, 3.0, 4.0])}
    float32 = rng.random() < 0.25
    heads, kv_heads, dim = rng.choice([(8, 4, 256), (16, 8, 256), (32, 16, 128), (16, 4, 128), (8, 2, 64), (16, 16, 64), (12, 4, 96)])
    n_groups = rng.choice([1, 1, 1, 2, 3])
    most = 24 if float32 else 128
    sizes, prefixes = [], []
    for _ in range(n_groups):
        sizes.append(_log_uniform(rng, 2, max(2, most // n_groups)))
        prefixes.append(PAGE * _log_uniform(rng, 1, (2048 if float32 else 16384) // PAGE // n_groups))
    window = rng.choice([0, 0, 0, 512, 4096])
    softcap = rng.choice([0.0, 50.0])
    return {"kind": "attention", "dtype": "float32" if float32 else "bfloat16", "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "v_dim": dim, "groups": ",".join(map(str, sizes)), "prefix": ",".join(map(str, prefixes)),
            "alone": rng.choice([0, 0, 1, 5]), "own": _log_uniform(rng, 1, 512), "window": window, "softcap": softcap,
            "sinks": rng.random() < 0.3}


# ---------------------------------------------------------------------------------------- inputs
def _ints(text):
    return [int(x) for x in text.split(",")]


def _layout(case):
    """([(first row, rows, shared positions)], rows): the groups of an attention case, then each request alone."""
    runs, at = [], 0
    for n, shared in zip(_ints(case["groups"]), _ints(case["prefix"])):
        runs.append((at, n, shared))
        at += n
    for _ in range(case["alone"]):
        runs.append((at, 1, 0))
        at += 1
    return runs, at


def _counts(case, seed):
    """Positions that each row has seen, its own included: what it shares and 1 to `own` positions."""
    runs, rows = _layout(case)
    rng = np.random.default_rng([seed, 1])
    counts = np.zeros(rows, np.int64)
    for row0, n, shared in runs:
        counts[row0 : row0 + n] = shared + rng.integers(max(1, case["own"] // 3), case["own"] + 1, size=n)
    return counts


def _prepare_attention(case, seed):
    device = torch.device("cuda")
    dtype = torch.float32 if case["dtype"] == "float32" else torch.bfloat16
    runs, rows = _layout(case)
    counts = _counts(case, seed)
    width = -(-int(counts.max()) // PAGE)
    rng = np.random.default_rng([seed, 2])
    total = sum(shared // PAGE + sum(-(-int(counts[r] - shared) // PAGE) for r in range(row0, row0 + n)) for row0, n, shared in runs)
    pages = rng.permutation(total).astype(np.int32)              # pages of a cache that has been in use lie in no order
    table = np.full((rows, width), -1, np.int32)
    share_id, share_len, at = np.zeros(rows, np.int32), np.zeros(rows, np.int32), 0
    for i, (row0, n, shared) in enumerate(runs):
        common = pages[at : at + shared // PAGE]
        at += shared // PAGE
        for r in range(row0, row0 + n):
            mine = -(-int(counts[r] - shared) // PAGE)
            table[r, : len(common)] = common
            table[r, len(common) : len(common) + mine] = pages[at : at + mine]
            at += mine
            share_id[r], share_len[r] = i, shared
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    k = torch.randn((total, case["kv_heads"], PAGE, case["dim"]), generator=g, device=device, dtype=torch.float32).to(dtype)
    v = torch.randn((total, case["kv_heads"], PAGE, case["v_dim"]), generator=g, device=device, dtype=torch.float32).to(dtype)
    q = (2.0 * torch.randn((rows, case["heads"], case["dim"]), generator=g, device=device, dtype=torch.float32)).to(dtype)
    sinks = torch.randn((case["heads"],), generator=g, device=device, dtype=torch.float32) if case["sinks"] else None
    on = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(device)
    return {"kind": "attention", "q": q, "k": k, "v": v, "sinks": sinks, "block_table": on(table), "row_count": on(counts),
            "share_id": on(share_id), "share_len": on(share_len), "window": case["window"] or None, "softcap": case["softcap"] or None,
            "scale": case["dim"] ** -0.5, "runs": runs, "counts": [int(c) for c in counts], "tables": table}


def _settings(case, seed):
    """(temperature, top_k, top_p, min_p, uniform) of every request; a top_k of 0, a top_p of 1 and a min_p of 0 filter nothing, a
    temperature of 0 takes the first largest logit."""
    rng = np.random.default_rng([seed, 3])
    rows = case["rows"]
    temperature = rng.choice([0.6, 0.7, 0.8, 1.0, 1.3], size=rows)
    top_k, top_p, min_p = np.zeros(rows, np.int32), np.ones(rows), np.zeros(rows)
    kinds = {"top_k": (1,), "top_p": (2,), "min_p": (4,), "top_k top_p": (3,), "mixed": (0, 1, 2, 3, 4, 5, 6, 7, 8)}[case["filters"]]
    for r in range(rows):
        kind = int(rng.choice(kinds))
        if kind == 8:
            temperature[r] = 0.0
            continue
        if kind & 1:
            top_k[r] = int(rng.choice([1, 20, 50, 64, 200, 1000]))
        if kind & 2:
            top_p[r] = float(rng.choice([0.5, 0.8, 0.9, 0.95, 0.99]))
        if kind & 4:
            min_p[r] = float(rng.choice([0.02, 0.05, 0.1, 0.3]))
    return temperature, top_k, top_p, min_p, rng.random(rows)


def _prepare_sampling(case, seed):
    device = torch.device("cuda")
    rows, vocab = case["rows"], case["vocab"]
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    logits = case["spread"] * torch.randn((rows, vocab), generator=g, device=device, dtype=torch.float32)
    likely = torch.randint(0, vocab, (rows, min(300, vocab)), generator=g, device=device)
    lift = 2.0 * case["spread"] + 3.0 * torch.empty(likely.shape, device=device).exponential_(1.0, generator=g)
    logits.scatter_reduce_(1, likely, lift, "amax")            # a token drawn twice takes the larger of its lifts
    logits = 30.0 * torch.tanh(logits / 30.0)                    # Gemma 2's soft cap over the logits
    temperature, top_k, top_p, min_p, uniform = _settings(case, seed)
    f64 = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.float64)).to(device)
    return {"kind": "sampling", "logits": logits, "temperature": f64(temperature), "top_k": torch.from_numpy(top_k).to(device),
            "top_p": f64(top_p), "min_p": f64(min_p), "uniform": f64(uniform)}


def prepare(case, seed):
    return _prepare_attention(case, seed) if case["kind"] == "attention" else _prepare_sampling(case, seed)


# ---------------------------------------------------------------------------------------- the passes
def _plain_attention(s):
    """Row by row: scores, their soft cap and mask, softmax with the sink, the weighted sum of the values; what a group shares is
    taken out of its pages once."""
    rows, heads, _ = s["q"].shape
    kv_heads, dv = s["k"].shape[1], s["v"].shape[3]
    q = s["q"].float().view(rows, kv_heads, heads // kv_heads, -1)
    out = torch.empty((rows, heads, dv), dtype=s["q"].dtype, device=s["q"].device)

    def lines(table, row, first, last):                          # positions first .. last of a row as [kv heads, positions, size] in 32 bits
        pages = s["block_table"][row, first // PAGE : -(-last // PAGE)].long()
        t = table[pages].permute(1, 0, 2, 3).reshape(kv_heads, -1, table.shape[3])
        return t[:, : last - first].float()

    def scores(row0, n, keys):                                   # [n, kv heads, heads a kv head, positions]
        x = torch.einsum("nkgd,kpd->nkgp", q[row0 : row0 + n], keys) * s["scale"]
        return s["softcap"] * torch.tanh(x / s["softcap"]) if s["softcap"] else x

    for row0, n, shared in s["runs"]:
        shared_v = lines(s["v"], row0, 0, shared) if shared else None
        shared_x = scores(row0, n, lines(s["k"], row0, 0, shared)) if shared else None
        for r in range(row0, row0 + n):
            count = s["counts"][r]
            x = scores(r, 1, lines(s["k"], r, shared, count))[0]
            v = lines(s["v"], r, shared, count)
            if shared:
                x = torch.cat([shared_x[r - row0], x], dim=-1)
            if s["window"] and count > s["window"]:
                x[..., : count - s["window"]] = -math.inf
            top = x.amax(dim=-1, keepdim=True)
            if s["sinks"] is not None:
                top = torch.maximum(top, s["sinks"].view(kv_heads, -1, 1))
            p = torch.exp(x - top)
            total = p.sum(dim=-1, keepdim=True)
            if s["sinks"] is not None:
                total = total + torch.exp(s["sinks"].view(kv_heads, -1, 1) - top)
            y = torch.einsum("kgp,kpd->kgd", p[..., shared:], v)
            if shared:
                y = y + torch.einsum("kgp,kpd->kgd", p[..., :shared], shared_v)
            out[r] = (y / total).reshape(heads, dv).to(out.dtype)
    return out


def _plain_sampling(s):
    """Everything in 64 bits: a request's cut through the sorted logits lies next to a border, and its draw is one number against a
    running total over the vocabulary."""
    logits = s["logits"].double()
    rows, vocab = logits.shape
    greedy = (s["temperature"] <= 0).view(-1, 1)
    x = logits / torch.where(greedy, torch.ones_like(s["temperature"]).view(-1, 1), s["temperature"].view(-1, 1))
    ordered, index = torch.sort(x, dim=1, descending=True, stable=True)          # ties go to the lowest index
    k = torch.where((s["top_k"] > 0) & (s["top_k"] < vocab), s["top_k"], vocab).long().view(-1, 1)
    keep = ordered >= ordered.gather(1, k - 1)                                   # what ties with the k-th stays
    e = torch.exp(ordered - ordered[:, :1]) * keep
    p = e / e.sum(dim=1, keepdim=True)
    before = torch.cumsum(p, dim=1) - p
    top_p = s["top_p"].view(-1, 1)
    keep &= (before < top_p) | (top_p >= 1.0)
    e = e * keep
    p = e / e.sum(dim=1, keepdim=True)
    keep &= p >= s["min_p"].view(-1, 1) * p[:, :1]
    e = torch.zeros_like(e).scatter_(1, index, e * keep)                         # back in the vocabulary's order
    running = torch.cumsum(e / e.sum(dim=1, keepdim=True), dim=1)
    passed = (running > s["uniform"].view(-1, 1)) & (e > 0)
    drawn = torch.where(passed.any(dim=1), passed.int().argmax(dim=1), vocab - 1 - (e > 0).flip(1).int().argmax(dim=1))
    return torch.where(greedy.view(-1), index[:, 0], drawn).int()


def run(state):
    s = state
    if not own:
        return _plain_attention(s) if s["kind"] == "attention" else _plain_sampling(s)
    from kapel_b200 import kernels as K

    if s["kind"] == "sampling":
        return K.sample_filtered(s["logits"], s["temperature"], s["top_k"], s["top_p"], s["min_p"], s["uniform"])
    return K.shared_prefix_attention(s["q"], s["k"], s["v"], s["block_table"], s["row_count"], s["share_id"], s["share_len"], PAGE,
                                     s["window"], s["scale"], s["softcap"], sinks=s["sinks"])


# ---------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["kind"] == "sampling":
        rows, vocab = case["rows"], case["vocab"]
        return {"bytes": 4 * rows * vocab + rows * (4 * 8 + 4 + 4), "flops": 3 * rows * vocab}
    counts = _counts(case, 0)                                    # other seeds' lengths come to nearly the same
    runs, rows = _layout(case)
    size = 4 if case["dtype"] == "float32" else 2
    d, dv, window = case["dim"], case["v_dim"], case["window"]
    read = seen = 0
    for row0, n, shared in runs:
        first = [max(0, int(c) - window) if window else 0 for c in counts[row0 : row0 + n]]
        read += max(0, shared - min(first))                      # shared positions that any of the group's rows sees
        for c, f in zip(counts[row0 : row0 + n], first):
            read += int(c) - max(f, shared)
            seen += int(c) - f
    return {"bytes": size * (read * case["kv_heads"] * (d + dv) + rows * case["heads"] * (d + dv)),
            "flops": 2 * seen * case["heads"] * (d + dv)}


# ---------------------------------------------------------------------------------------- the definition in 64 bits
def _exact_attention(case, seed):
    s = _prepare_attention(case, seed)
    rows, heads, d = s["q"].shape
    kv_heads = s["k"].shape[1]
    out = torch.empty((rows, heads, s["v"].shape[3]), dtype=torch.float64)
    device = s["q"].device
    for r in range(rows):
        count = s["counts"][r]
        first = max(0, count - s["window"]) if s["window"] else 0
        at = torch.arange(first, count)
        pages = torch.from_numpy(s["tables"][r].astype(np.int64))[at // PAGE].to(device)
        keys, values = s["k"][pages, :, (at % PAGE).to(device)].double(), s["v"][pages, :, (at % PAGE).to(device)].double()
        for h in range(kv_heads):
            of = slice(h * (heads // kv_heads), (h + 1) * (heads // kv_heads))
            x = s["q"][r, of].double() @ keys[:, h].T * s["scale"]
            if s["softcap"]:
                x = torch.tanh(x / s["softcap"]) * s["softcap"]
            if s["sinks"] is not None:                           # a key of that score whose value is zero
                x = torch.cat([x, s["sinks"][of].double().view(-1, 1)], dim=1)
            w = torch.softmax(x, dim=1)[:, : count - first]
            out[r, of] = (w @ values[:, h]).cpu()
    return out


def _exact_sampling(case, seed):
    s = _prepare_sampling(case, seed)
    host = s["logits"].cpu().numpy()
    temperature, top_k, top_p, min_p, uniform = _settings(case, seed)
    tokens = np.zeros(case["rows"], np.int32)
    for r in range(case["rows"]):
        row = host[r].astype(np.float64)
        if temperature[r] <= 0:
            tokens[r] = int(np.argmax(row))
            continue
        row = row / temperature[r]
        alive = np.arange(row.size)
        if 0 < top_k[r] < row.size:
            alive = alive[row >= np.partition(row, row.size - int(top_k[r]))[row.size - int(top_k[r])]]
        weight = np.exp(row[alive] - row.max())
        if top_p[r] < 1.0:
            order = np.argsort(-row[alive], kind="stable")
            total = np.cumsum(weight[order])
            n = int(np.searchsorted(total, top_p[r] * total[-1], side="left")) + 1       # the first whose total reaches it, and all before
            kept = np.sort(order[:n])
            alive, weight = alive[kept], weight[kept]
        above = weight >= min_p[r] * weight.max()
        alive, weight = alive[above], weight[above]
        total = np.cumsum(weight)
        tokens[r] = alive[min(int(np.searchsorted(total, uniform[r] * total[-1], side="right")), alive.size - 1)]
    return torch.from_numpy(tokens)


def exact(case, seed):
    return _exact_attention(case, seed) if case["kind"] == "attention" else _exact_sampling(case, seed)
