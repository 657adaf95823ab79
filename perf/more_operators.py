"""What a recurrent language model needs in front of, between and behind its layers, as measurable cases: the embedding of tokens
with its gradient, a gated linear recurrence over long sequences (prompts, training, single tokens), and beam search's
selection with the reordering of the states that beams carry.  Each in its plain form (elementary torch operations in 32 bits) and as
the framework's own entry points.

A case is a dict of plain values.  `op` names the operator, `call` what is done with it:
  embed     `tokens` rows of a table of vocabulary x width, of type `table`, as activations of type `dtype`; "forward" or "train"
  recur     `sequences` of at most `longest` tokens (`packed`: of lengths of their own, one behind the other; else all of that length),
            `width` channels, `gate`: with an output gate; "forward" or "train"
  tick      one token each of `sequences`, the state updated in place
  select    `beams` of each of `sequences` continued over `vocabulary`
  reorder   the states of the beams moved behind a selection: an LSTM's h and c of `width` and a memory of heads x d x d, fp32
"""
import math
import random

import torch

own = False

_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_SIZE = {"f16": 2, "bf16": 2, "f32": 4}


def listed():
    return [
        # the embedding of a token each while 32 sequences are served
        dict(name="embed_token", op="embed", call="forward", tokens=32, vocabulary=32000, width=1024, table="f32", dtype="f16", scale=1.0),
        # a training step's embedding and its gradient, fp32 parameters, a vocabulary that is a multiple of nothing
        dict(name="embed_train", op="embed", call="train", tokens=65536, vocabulary=50001, width=1024, table="f32", dtype="f16", scale=1.0),
        # a small model, all fp32, a width that is a multiple of nothing, scaled by the root of the width (200 steps of 70 rows)
        dict(name="embed_train_ragged_f32", op="embed", call="train", tokens=14000, vocabulary=1000, width=257, table="f32", dtype="f32",
             scale=257 ** 0.5),
        # one sequence, one token: latency alone
        dict(name="tick_one", op="tick", call="tick", sequences=1, width=1024, gate=True, dtype="f16"),
        # a large batch being served, a token each
        dict(name="tick_batch", op="tick", call="tick", sequences=2048, width=5120, gate=True, dtype="bf16"),
        # the headline configuration's activations (256 sequences of 1024 steps of 1024 channels), trained
        dict(name="recur_train", op="recur", call="train", sequences=256, longest=1024, packed=False, width=1024, gate=True, dtype="f16"),
        # one very long prompt: the work lies along the sequence
        dict(name="recur_prompt_long", op="recur", call="forward", sequences=1, longest=131072, packed=False, width=1024, gate=True, dtype="bf16"),
        # packed sequences of odd sizes on fp32 tensors, trained
        dict(name="recur_train_ragged_f32", op="recur", call="train", sequences=7, longest=2000, packed=True, width=257, gate=False, dtype="f32"),
        # one user's search
        dict(name="select_one", op="select", call="select", sequences=1, beams=4, vocabulary=32000, dtype="f16"),
        # a batch of searches, a vocabulary that is a multiple of nothing
        dict(name="select_batch", op="select", call="select", sequences=64, beams=8, vocabulary=50001, dtype="bf16"),
        # the states behind one user's selection
        dict(name="reorder_one", op="reorder", call="reorder", sequences=1, beams=4, width=1024, heads=16, d=64),
        # the states behind a batch's selection
        dict(name="reorder_batch", op="reorder", call="reorder", sequences=64, beams=8, width=1024, heads=16, d=64),
    ]


def _between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: sizes over the whole range by their logarithm, half of them round numbers and half of them not."""
    op = rng.choice(["embed", "embed", "embed", "recur", "recur", "recur", "recur", "tick", "select", "select", "reorder"])
    dtype, even = rng.choice(list(_TYPES)), rng.random() < 0.5
    width = _between(rng, 32, 8192)
    width = max(32, width // 32 * 32) if even else width
    if op == "embed":
        vocabulary = _between(rng, 1000, 262144)
        case = dict(op=op, call=rng.choice(["forward", "train", "train"]), tokens=_between(rng, 1, 262144),
                    vocabulary=vocabulary // 64 * 64 if even else vocabulary, width=width, table=rng.choice(["f32", dtype]), dtype=dtype,
                    scale=rng.choice([1.0, width ** 0.5]))
        while 4 * (case["tokens"] + vocabulary) * case["width"] > 1e9:
            case["width"] = max(32, case["width"] // 2)
            case["tokens"] = max(1, case["tokens"] * 3 // 4)
        return case
    if op in ("recur", "tick"):
        case = dict(op=op, call=op, sequences=_between(rng, 1, 256 if op == "recur" else 2048), width=width, gate=rng.random() < 0.5, dtype=dtype)
        if op == "recur":
            case.update(call=rng.choice(["forward", "train"]), longest=_between(rng, 1, 65536), packed=rng.random() < 0.5)
            while case["sequences"] * case["longest"] * width > 1 << 26:
                if rng.random() < 0.5 and case["sequences"] > 1:
                    case["sequences"] //= 2
                else:
                    case["longest"] = max(1, case["longest"] // 2)
        return case
    sequences, beams = _between(rng, 1, 256), _between(rng, 2, 16)
    if op == "reorder":
        case = dict(op=op, call=op, sequences=sequences, beams=beams, width=width, heads=rng.choice([1, 4, 16]), d=rng.choice([16, 64, 128, 33]))
        while beams * case["sequences"] * case["heads"] * case["d"] ** 2 > 1 << 28:
            case["sequences"] //= 2
        return case
    vocabulary = _between(rng, 1000, 131072)
    vocabulary = vocabulary // 64 * 64 if even else vocabulary
    return dict(op=op, call=op, sequences=max(1, min(sequences, 400000000 // (beams * vocabulary * _SIZE[dtype]))), beams=beams, vocabulary=vocabulary,
                dtype=dtype)


def _lengths(case):
    """The sequences' lengths: whole ones, or for packed sequences ones that the case alone decides, the longest and one of a
    single token among them."""
    n, longest = case["sequences"], case["longest"]
    if not case["packed"]:
        return [longest] * n
    r = random.Random(n * 1000003 + longest)
    return ([longest, 1] + [max(1, int(longest * r.random())) for _ in range(n)])[:n]


def _parents(case, seed):
    """The beams that a selection continues: in the order of the new scores, good ones more than once, some not at all, and in
    some sequences all of them as they were."""
    r, beams = random.Random(seed), case["beams"]
    return [list(range(beams)) if r.random() < 0.25 else [int(beams * r.random() ** 2) for _ in range(beams)] for _ in range(case["sequences"])]


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, device=dev, generator=g, dtype=torch.float32).to(dtype)

    def uniform(*shape):
        return torch.rand(*shape, device=dev, generator=g)

    s = dict(case=case)
    if case["op"] == "embed":
        tokens, vocabulary, width = case["tokens"], case["vocabulary"], case["width"]
        # tokens of a text: the n-th most frequent with a share of about 1 / n, wherever it stands in the table; some padding
        rank = (torch.exp(uniform(tokens) * math.log(vocabulary + 1)).long() - 1).clamp(0, vocabulary - 1)
        s["tokens"] = torch.where(uniform(tokens) < 1 / 64, -1, rank * 7919 % vocabulary)
        s["table"] = normal(vocabulary, width, dtype=_TYPES[case["table"]])
        if case["call"] == "train":
            s["d_out"] = normal(tokens, width, dtype=_TYPES[case["dtype"]])
        return s
    if case["op"] in ("recur", "tick"):
        dtype, n, width = _TYPES[case["dtype"]], case["sequences"], case["width"]
        s["lengths"] = lengths = _lengths(case) if case["op"] == "recur" else [1] * n
        if case["op"] == "tick":
            shape = (n,)
        else:
            shape = (sum(lengths),) if case["packed"] else (n, case["longest"])
            s["cu_seqlens"] = torch.tensor([0] + lengths, device=dev).cumsum(0).to(torch.int32) if case["packed"] else None
        # x, forget and gate as one projection gives them, beside each other in a row; memories of 2 to some 500 tokens
        rows = normal(*shape, (3 if case["gate"] else 2) * width, dtype=dtype)
        parts = rows.split(width, -1)
        parts[1].add_((6 * uniform(width)).to(dtype))
        s["x"], s["forget"], s["gate"] = parts[0], parts[1], parts[2] if case["gate"] else None
        s["state"] = normal(n, width)
        if case["call"] == "train":
            s["dy"], s["d_state"] = normal(*shape, width, dtype=dtype), normal(n, width)
        return s
    n, beams = case["sequences"], case["beams"]
    if case["op"] == "reorder":
        s["parents"] = torch.tensor(_parents(case, seed), device=dev, dtype=torch.int64)
        s["states"] = [normal(n * beams, case["width"], dtype=torch.float16), normal(n * beams, case["width"], dtype=torch.float16),
                       normal(n * beams, case["heads"], case["d"], case["d"])]
        return s
    s["logits"] = normal(n, beams, case["vocabulary"], dtype=_TYPES[case["dtype"]]).mul_(2.5)
    s["logits"][..., 0] = -math.inf                                  # (a token that must not come)
    s["scores"] = -torch.sort(20 * uniform(n, beams), -1).values
    s["scores"][0, 1:] = -math.inf                                   # the first sequence begins its search: one beam alone
    s["finished"] = uniform(n, beams) < 1 / 16
    s["finished"][0] = False
    s["end"] = 1
    return s


# ---- the framework's entry points

def _run_own(s):
    import flashlstm_poc_amd as fl
    case = s["case"]
    op, train = case["op"], case["call"] == "train"
    if op == "embed":
        dtype, table = _TYPES[case["dtype"]], _TYPES[case["table"]]
        out = dict(out=fl.embedding_forward(s["tokens"], s["table"], scale=case["scale"], dtype=dtype))
        if train:
            out["d_table"] = fl.embedding_backward(s["d_out"], s["tokens"], case["vocabulary"], scale=case["scale"], dtype=table)
        return out
    if op == "tick":
        return dict(y=fl.gated_recurrence_step(s["x"], s["forget"], s["state"], s["gate"]), state=s["state"])
    if op == "recur":
        y, state, saved = fl.gated_recurrence_forward(s["x"], s["forget"], s["gate"], state=s["state"], cu_seqlens=s["cu_seqlens"], want_saved=train)
        out = dict(y=y, state=state)
        if train:
            out["dx"], out["dforget"], out["dgate"], out["d_initial"] = fl.gated_recurrence_backward(
                s["dy"], s["x"], s["forget"], s["gate"], saved, d_state=s["d_state"], cu_seqlens=s["cu_seqlens"])
        return out
    if op == "select":
        scores, parents, tokens, finished = fl.beam_select(s["logits"], s["scores"], end=s["end"], finished=s["finished"])
        return dict(scores=scores, parents=parents, tokens=tokens, finished=finished)
    fl.beam_reorder(s["parents"], *s["states"])
    return s["states"]


# ---- the plain forms

def _embed_plain(s):
    case, table = s["case"], s["table"]
    held = (s["tokens"] >= 0) & (s["tokens"] < case["vocabulary"])
    index = torch.where(held, s["tokens"], 0)
    out = dict(out=torch.where(held[:, None], case["scale"] * table[index].float(), 0.0).to(_TYPES[case["dtype"]]))
    if case["call"] == "train":
        d = torch.where(held[:, None], s["d_out"].float(), 0.0)
        sums = torch.zeros(table.shape, device=table.device, dtype=torch.float32).index_add_(0, index, d)
        out["d_table"] = (case["scale"] * sums).to(table.dtype)
    return out


def _sigmoid(x):
    return 1 / (1 + torch.exp(-x))


def _tick_plain(s):
    x, forget, dtype = s["x"].float(), s["forget"].float(), s["x"].dtype
    c = _sigmoid(forget) * s["state"] + _sigmoid(-forget) * x
    s["state"].copy_(c)
    return dict(y=(c if s["gate"] is None else _sigmoid(s["gate"].float()) * c).to(dtype), state=s["state"])


def _walk(f, b, first):
    """h_t = f_t h_{t-1} + b_t over axis 1 of (n, L, width) from `first` (n, width): pieces of about the root of L tokens walked side by
    side, each with the product of its factors, then one behind the other."""
    n, length, width = f.shape
    piece = max(1, math.isqrt(length))
    count = -(-length // piece)
    if count * piece != length:
        more = (n, count * piece - length, width)
        f, b = torch.cat([f, f.new_ones(more)], 1), torch.cat([b, b.new_zeros(more)], 1)
    f, b = f.view(n, count, piece, width), b.view(n, count, piece, width)
    h, product = torch.empty_like(b), torch.empty_like(f)
    h[:, :, 0], product[:, :, 0] = b[:, :, 0], f[:, :, 0]
    for i in range(1, piece):
        torch.addcmul(b[:, :, i], f[:, :, i], h[:, :, i - 1], out=h[:, :, i])
        torch.mul(f[:, :, i], product[:, :, i - 1], out=product[:, :, i])
    for j in range(count):
        h[:, j].addcmul_(product[:, j], first[:, None])
        first = h[:, j, -1]
    return h.view(n, count * piece, width)[:, :length]


def _recur_plain(s):
    lengths, dtype, dev = s["lengths"], s["x"].dtype, s["x"].device
    n, longest, width = len(lengths), max(lengths), s["case"]["width"]
    length = torch.tensor(lengths, device=dev)
    at = torch.arange(longest, device=dev)
    inside = at < length[:, None]                                               # (n, longest)
    row = torch.where(inside, (length.cumsum(0) - length)[:, None] + at, 0)
    whole = not s["case"]["packed"]

    def spread(t):    # the caller's layout -> (n, longest, width) in 32 bits
        return t.float() if whole else t.float()[row]

    def gather(t):
        return (t if whole else t[inside]).to(dtype)

    def masked(t):    # zeros behind a sequence's end
        return t if whole else t * inside[..., None]

    x, u = spread(s["x"]), spread(s["forget"])
    f, z = _sigmoid(u), masked(_sigmoid(-u))
    if not whole:
        f = torch.where(inside[..., None], f, 1.0)
    c = _walk(f, z * x, s["state"])
    o = None if s["gate"] is None else _sigmoid(spread(s["gate"]))
    out = dict(y=gather(c if o is None else o * c), state=c[:, -1].clone())
    if s["case"]["call"] == "train":
        dy = masked(spread(s["dy"]))
        dc = dy if o is None else dy * o
        # G_t = dc_t + f_{t+1} G_{t+1}, from the last token to the first: with H_t = f_t G_t, H_t = f_t H_{t+1} + f_t dc_t
        flipped = _walk(f.flip(1), (f * dc).flip(1), s["d_state"]).flip(1)      # H
        total = dc + torch.cat([flipped[:, 1:], s["d_state"][:, None]], 1)      # G
        before = torch.cat([s["state"][:, None], c[:, :-1]], 1)
        out["dx"] = gather(z * total)
        out["dforget"] = gather(total * (before - x) * f * z)
        out["dgate"] = None if o is None else gather(dy * c * o * (1 - o))
        out["d_initial"] = flipped[:, 0].clone()
    return out


def _select_plain(s):
    """(Candidates in 64 bits: which is larger must not depend on a rounding of their sums.)"""
    n, beams, vocabulary = s["logits"].shape
    z = s["logits"].double()
    most = z.amax(-1, keepdim=True)
    value = z - most - torch.log(torch.exp(z - most).sum(-1, keepdim=True)) + s["scores"].double()[..., None]
    done = s["finished"][..., None]
    value = torch.where(done, -math.inf, value)
    value[..., s["end"]] = torch.where(s["finished"], s["scores"].double(), value[..., s["end"]])
    value = value.view(n, beams * vocabulary)
    scores, places = [], []
    for _ in range(beams):
        best = value.amax(-1, keepdim=True)
        place = (value == best).to(torch.int8).argmax(-1, keepdim=True)        # the lowest of equal ones
        scores.append(best)
        places.append(place)
        value.scatter_(1, place, -math.inf)
    scores, places = torch.cat(scores, 1), torch.cat(places, 1)
    parents, tokens = places // vocabulary, places % vocabulary
    return dict(scores=scores.float(), parents=parents, tokens=tokens, finished=tokens == s["end"])


def _reorder_plain(s):
    n, beams = s["parents"].shape
    rows = (s["parents"] + beams * torch.arange(n, device=s["parents"].device)[:, None]).flatten()
    for state in s["states"]:
        state.copy_(state[rows])
    return s["states"]


def run(s):
    if own:
        return _run_own(s)
    return {"embed": _embed_plain, "tick": _tick_plain, "recur": _recur_plain, "select": _select_plain, "reorder": _reorder_plain}[s["case"]["op"]](s)


def _distinct(tokens, vocabulary):
    """How many of the vocabulary's tokens a text of `tokens` is expected to hold (as `prepare` draws them)."""
    edge = torch.log(torch.arange(1, vocabulary + 2, dtype=torch.float64)) / math.log(vocabulary + 1)
    share = (edge[1:] - edge[:-1]) * (63 / 64)
    return float((1 - (1 - share) ** tokens).sum())


def work(case):
    """Bytes: every input once, every output once; of a table the rows that the text holds, of states the rows that move.  Operations: a
    product and a sum a value, of the recurrence the gates' exponentials and quotients too, of the selection an exponential and a sum."""
    op, train = case["op"], case["call"] == "train"
    if op == "embed":
        tokens, width = case["tokens"], case["width"]
        rows, one = tokens * width, _SIZE[case["table"]]
        size = 8 * tokens + rows * _SIZE[case["dtype"]] + _distinct(tokens, case["vocabulary"]) * width * one
        if train:
            size += rows * _SIZE[case["dtype"]] + case["vocabulary"] * width * one
        return {"bytes": float(size), "flops": float(rows * (2 if train else 1))}
    if op in ("recur", "tick"):
        e, tokens = _SIZE[case["dtype"]], sum(_lengths(case)) if op == "recur" else case["sequences"]
        n, tensors = tokens * case["width"], (4 if case["gate"] else 3) * (2 if train else 1)
        states = 8 * case["sequences"] * case["width"] * (2 if train else 1)
        return {"bytes": float(states + e * n * tensors), "flops": (40.0 if train else 12.0) * n}
    if op == "select":
        n = case["sequences"] * case["beams"] * case["vocabulary"]
        return {"bytes": float(n * _SIZE[case["dtype"]] + case["sequences"] * case["beams"] * 26), "flops": 4.0 * n}
    moved = sum(len({p for i, p in enumerate(row) if p != i}) + sum(p != i for i, p in enumerate(row)) for row in _parents(case, 0))
    return {"bytes": float(8 * case["sequences"] * case["beams"] + moved * (4 * case["width"] + 4 * case["heads"] * case["d"] ** 2)), "flops": 0.0}


# ---- the definitions in 64 bits

def _embed_exact(s):
    case, tokens, scale = s["case"], s["tokens"], s["case"]["scale"]
    table = torch.cat([s["table"].double(), torch.zeros(1, case["width"], device=tokens.device, dtype=torch.float64)])
    places = tokens.masked_fill((tokens < 0) | (tokens >= case["vocabulary"]), case["vocabulary"])   # the row behind the last holds zeros
    out = dict(out=scale * torch.nn.functional.embedding(places, table))
    if case["call"] == "train":
        order = torch.argsort(places, stable=True)
        counts = torch.bincount(places, minlength=case["vocabulary"] + 1)
        ends = counts.cumsum(0)
        sums = torch.zeros_like(table)
        # (columns at a time: the running sum over all tokens of a part of them, and its differences at the tokens' borders)
        for columns in torch.arange(case["width"], device=tokens.device).split(128):
            running = torch.cat([torch.zeros(1, len(columns), device=tokens.device, dtype=torch.float64), s["d_out"][:, columns].double()[order].cumsum(0)])
            sums[:, columns] = running[ends] - running[ends - counts]
        out["d_table"] = scale * sums[:-1]
    return out


def _tick_exact(s):
    f = torch.sigmoid(s["forget"].double())
    c = torch.lerp(s["x"].double(), s["state"].double(), f)
    return dict(y=c if s["gate"] is None else torch.sigmoid(s["gate"].double()) * c, state=c)


def _recur_exact(s):
    """Token by token, all sequences that are that long; backwards the same."""
    case, lengths, train = s["case"], s["lengths"], s["case"]["call"] == "train"
    packed, dev = case["packed"], s["x"].device
    starts = [sum(lengths[:i]) for i in range(len(lengths))] if packed else [i * case["longest"] for i in range(len(lengths))]
    # sequences by falling length, so that those with a token t are the first ones
    by = sorted(range(len(lengths)), key=lambda i: -lengths[i])
    first = torch.tensor([starts[i] for i in by], device=dev)
    order = torch.tensor(by, device=dev)
    alive, k = [], len(by)
    for t in range(max(lengths)):
        while lengths[by[k - 1]] <= t:
            k -= 1
        alive.append(k)
    flat = {name: None if s.get(name) is None else s[name].reshape(-1, case["width"]) for name in ("x", "forget", "gate", "dy")}
    c = s["state"].double()[order]
    kept = torch.empty(len(flat["x"]), case["width"], device=dev, dtype=torch.float64)
    for t, k in enumerate(alive):
        rows = first[:k] + t
        f = torch.sigmoid(flat["forget"][rows].double())
        c[:k] = torch.lerp(flat["x"][rows].double(), c[:k], f)
        kept[rows] = c[:k]
    state = torch.empty_like(c)
    state[order] = c
    shape = s["x"].shape
    out = dict(y=(kept if flat["gate"] is None else kept * torch.sigmoid(flat["gate"].double())).view(shape), state=state)
    if not train:
        return out
    dx, dforget = torch.empty_like(kept), torch.empty_like(kept)
    dgate = None if flat["gate"] is None else torch.empty_like(kept)
    total, start = s["d_state"].double()[order], s["state"].double()[order]
    for t in range(len(alive) - 1, -1, -1):
        k = alive[t]
        rows = first[:k] + t
        f, dy = torch.sigmoid(flat["forget"][rows].double()), flat["dy"][rows].double()
        if dgate is not None:
            o = torch.sigmoid(flat["gate"][rows].double())
            dgate[rows] = dy * kept[rows] * o * (1 - o)
            dy = dy * o
        total[:k] += dy
        before = kept[rows - 1] if t > 0 else start[:k]
        z = torch.sigmoid(-flat["forget"][rows].double())
        dx[rows] = total[:k] * z
        dforget[rows] = total[:k] * (before - flat["x"][rows].double()) * f * z
        total[:k] *= f
    initial = torch.empty_like(total)
    initial[order] = total
    out.update(dx=dx.view(shape), dforget=dforget.view(shape), dgate=None if dgate is None else dgate.view(shape), d_initial=initial)
    return out


def _select_exact(s):
    n, beams, vocabulary = s["logits"].shape
    parts = []
    for i in range(n):   # (a sequence at a time: 64 bits of them all are large)
        log_p = torch.log_softmax(s["logits"][i].double(), -1) + s["scores"][i].double()[:, None]
        log_p[s["finished"][i]] = -math.inf
        rows = s["finished"][i].nonzero().flatten()
        log_p[rows, s["end"]] = s["scores"][i, rows].double()
        best, place = torch.sort(log_p.flatten(), descending=True, stable=True)
        parts.append((best[:beams], place[:beams]))
    scores, places = (torch.stack(p) for p in zip(*parts))
    tokens = places.remainder(vocabulary)
    return dict(scores=scores, parents=torch.div(places, vocabulary, rounding_mode="floor"), tokens=tokens, finished=tokens.eq(s["end"]))


def _reorder_exact(s):
    out = []
    for state in s["states"]:
        by_sequence = state.double().unflatten(0, s["parents"].shape)
        out.append(torch.stack([rows[p] for rows, p in zip(by_sequence, s["parents"])]).flatten(0, 1))
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"embed": _embed_exact, "tick": _tick_exact, "recur": _recur_exact, "select": _select_exact, "reorder": _reorder_exact}[case["op"]](s)
