"""The operators that a recurrent language model needs around its LSTM layers, as measurable cases: layer norm on a residual
stream, attention whose memory is a decaying state of fixed size (prompts, training, single tokens), and the distillation
loss against a teacher's top logits.  Each in its plain form (elementary torch operations in 32 bits) and as the framework's
own entry points.

A case is a dict of plain values.  `op` names the operator, `call` what is done with it:
  norm     rows x width; "forward", or "train" (forward and backward)
  attend   `sequences` of at most `longest` tokens (`packed`: of lengths of their own, one behind the other; else all of that
           length), `heads` of queries and `kv_heads` of keys and values, `dk` x `dv` a head; "forward" or "train"
  step     one token each of `sequences`, the state updated in place
  distill  rows x vocabulary, `top` teacher entries a row; "forward", or "train" (loss and gradient in one call), or "both"
           (loss first, gradient in a call of its own)
"""
import math
import random

import torch

own = False

_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_SIZE = {"f16": 2, "bf16": 2, "f32": 4}


def listed():
    return [
        # the norm in front of a layer while 32 sequences are served, a token each
        dict(name="norm_token", op="norm", call="forward", rows=32, width=1024, dtype="f16", residual=True),
        # a training step's norm over the activations of the headline configuration (1024 steps of 256 rows of 1024)
        dict(name="norm_train", op="norm", call="train", rows=262144, width=1024, dtype="f16", residual=True),
        # a small model of a width that is a multiple of nothing, trained on fp32 tensors (200 steps of 70 rows)
        dict(name="norm_train_ragged_f32", op="norm", call="train", rows=14000, width=257, dtype="f32", residual=False),
        # one sequence, one token: latency alone
        dict(name="step_one", op="step", call="step", sequences=1, heads=16, kv_heads=16, dk=64, dv=64, dtype="f16"),
        # a batch being served, a token each: the states are read and written once
        dict(name="step_batch", op="step", call="step", sequences=256, heads=16, kv_heads=4, dk=128, dv=128, dtype="bf16"),
        # prompts of different lengths, packed, heads that share keys and values
        dict(name="prompt_packed", op="attend", call="forward", sequences=12, longest=4096, packed=True, heads=16, kv_heads=4,
             dk=128, dv=128, dtype="bf16"),
        # one very long prompt: few rows, the work lies along the sequence
        dict(name="prompt_long", op="attend", call="forward", sequences=1, longest=131072, packed=False, heads=8, kv_heads=8,
             dk=128, dv=128, dtype="f16"),
        # a training step's attention (16 sequences of 2048 tokens, 2048 features)
        dict(name="attend_train", op="attend", call="train", sequences=16, longest=2048, packed=False, heads=16, kv_heads=16,
             dk=128, dv=128, dtype="bf16"),
        # packed sequences of odd sizes on fp32 tensors, heads that share keys and values
        dict(name="attend_train_ragged_f32", op="attend", call="train", sequences=7, longest=200, packed=True, heads=6, kv_heads=2,
             dk=40, dv=65, dtype="f32"),
        # a small batch's loss and gradient, fp32 logits, two calls as autograd makes them
        dict(name="distill_small_f32", op="distill", call="both", rows=32, vocabulary=32000, top=8, dtype="f32"),
        # scoring held-out text against the teacher
        dict(name="distill_score", op="distill", call="forward", rows=2048, vocabulary=32000, top=32, dtype="f16"),
        # a training step's loss and gradient, a vocabulary that is a multiple of nothing
        dict(name="distill_train", op="distill", call="train", rows=8192, vocabulary=50001, top=64, dtype="bf16"),
    ]


def _between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: sizes over the whole range by their logarithm, half of them round numbers and half of them not."""
    op, dtype, even = rng.choice(["norm", "norm", "attend", "attend", "attend", "step", "distill", "distill"]), rng.choice(list(_TYPES)), rng.random() < 0.5
    if op == "norm":
        rows, width = _between(rng, 1, 262144), _between(rng, 32, 8192)
        width = max(32, width // 32 * 32) if even else width
        return dict(op=op, call=rng.choice(["forward", "train"]), rows=max(1, min(rows, (1 << 29) // (width * _SIZE[dtype]))), width=width, dtype=dtype,
                    residual=rng.random() < 0.5)
    if op == "distill":
        rows, vocabulary = _between(rng, 1, 8192), _between(rng, 1000, 131072)
        vocabulary = vocabulary // 64 * 64 if even else vocabulary
        return dict(op=op, call=rng.choice(["forward", "train", "both"]), rows=max(1, min(rows, 800000000 // (vocabulary * _SIZE[dtype]))), vocabulary=vocabulary,
                    top=_between(rng, 1, 256), dtype=dtype)
    dk, dv = (rng.choice([32, 64, 128, 256]), rng.choice([32, 64, 128, 256])) if even else (_between(rng, 16, 256), _between(rng, 16, 256))
    kv_heads = rng.choice([1, 2, 4, 8])
    case = dict(op=op, call="step", sequences=_between(rng, 1, 256), heads=kv_heads * rng.choice([1, 1, 2, 4]), kv_heads=kv_heads, dk=dk, dv=dv,
                dtype=dtype)
    if op == "step":
        while work(case)["bytes"] > 1e9:
            case["sequences"] //= 2
        return case
    case.update(call=rng.choice(["forward", "train"]), longest=_between(rng, 1, 65536), packed=rng.random() < 0.5)
    case["sequences"] = min(case["sequences"], 64)
    while work(case)["bytes"] > 5e8 or case["longest"] * case["sequences"] * case["heads"] > 1 << 20:
        case["longest"] = max(1, case["longest"] // 2)
        case["sequences"] = case["sequences"] if case["longest"] > 16 else max(1, case["sequences"] // 2)
    return case


def _lengths(case):
    """The sequences' lengths: whole ones, or for packed sequences ones that the case alone decides, the longest and one of a
    single token among them."""
    n, longest = case["sequences"], case["longest"]
    if not case["packed"]:
        return [longest] * n
    r = random.Random(n * 1000003 + longest)
    return ([longest, 1] + [max(1, int(longest * r.random())) for _ in range(n)])[:n]


def prepare(case, seed):
    dev, dtype = "cuda", _TYPES[case["dtype"]]
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, dtype=dtype):
        return torch.randn(*shape, device=dev, generator=g, dtype=torch.float32).to(dtype)

    s = dict(case=case)
    if case["op"] == "norm":
        rows, width = case["rows"], case["width"]
        s["x"] = torch.add(normal(rows, width), normal(rows, 1) * 0.5)
        s["residual"] = normal(rows, width) if case["residual"] else None
        s["weight"], s["bias"] = 1 + 0.1 * normal(width, dtype=torch.float32), 0.1 * normal(width, dtype=torch.float32)
        if case["call"] == "train":
            s["dy"] = normal(rows, width)
            s["d_total"] = normal(rows, width) if case["residual"] else None
        return s
    if case["op"] == "distill":
        rows, vocabulary, top = case["rows"], case["vocabulary"], case["top"]
        s["logits"] = normal(rows, vocabulary).mul_(2.5)
        s["teacher_logits"] = torch.sort(normal(rows, top, dtype=torch.float32) * 2 + 8, descending=True).values
        # distinct tokens: an offset and a stride of each row's own; the tail of some lists is empty, and rows of padding are
        start = torch.randint(0, vocabulary, (rows, 1), device=dev, generator=g)
        stride = torch.randint(1, max(2, vocabulary // top), (rows, 1), device=dev, generator=g)
        index = (start + stride * torch.arange(top, device=dev)) % vocabulary
        kept = torch.randint(max(1, top // 2), top + 1, (rows, 1), device=dev, generator=g)
        kept = torch.where(torch.rand(rows, 1, device=dev, generator=g) < 1 / 16, torch.zeros_like(kept), kept)
        kept[0] = top
        s["teacher_index"] = torch.where(torch.arange(top, device=dev) < kept, index, -1).to(torch.int32)
        s["temperature"] = 2.0
        s["d_loss"] = torch.rand(rows, device=dev, generator=g) / rows
        return s
    heads, kv, dk, dv, n = case["heads"], case["kv_heads"], case["dk"], case["dv"], case["sequences"]
    # a memory of 4 to 256 tokens, longer from head to head
    s["log_decay"] = torch.log1p(-torch.exp2(-torch.linspace(2, 8, heads, device=dev) - 0.1 * torch.rand(heads, device=dev, generator=g)))
    s["state"] = normal(n, heads, dk, dv, dtype=torch.float32)
    if case["op"] == "step":
        s["q"], s["k"], s["v"] = normal(n, heads, dk), normal(n, kv, dk), normal(n, kv, dv)
        return s
    lengths = _lengths(case)
    s["lengths"] = lengths
    shape = (sum(lengths),) if case["packed"] else (n, case["longest"])
    s["cu_seqlens"] = torch.tensor([0] + lengths, device=dev).cumsum(0).to(torch.int32) if case["packed"] else None
    s["q"], s["k"], s["v"] = normal(*shape, heads, dk), normal(*shape, kv, dk), normal(*shape, kv, dv)
    if case["call"] == "train":
        s["do"], s["d_state"] = normal(*shape, heads, dv), normal(n, heads, dk, dv, dtype=torch.float32)
    return s


# ---- the framework's entry points

def _run_own(s):
    import flashlstm_poc_amd as fl
    case = s["case"]
    op, train = case["op"], case["call"] == "train"
    if op == "norm":
        y, total, mean, rstd = fl.layer_norm_forward(s["x"], s["weight"], s["bias"], residual=s["residual"])
        out = dict(y=y, total=total if case["residual"] else None)
        if train:
            out["dx"], out["dweight"], out["dbias"] = fl.layer_norm_backward(s["dy"], total, s["weight"], mean, rstd, d_total=s["d_total"])
        return out
    if op == "distill":
        teacher = (s["teacher_logits"], s["teacher_index"])
        if train:
            loss, dlogits = fl.distillation_train(s["logits"], *teacher, s["d_loss"], temperature=s["temperature"])
            return dict(loss=loss, dlogits=dlogits)
        loss, lse = fl.distillation_forward(s["logits"], *teacher, temperature=s["temperature"])
        if case["call"] == "forward":
            return dict(loss=loss)
        return dict(loss=loss, dlogits=fl.distillation_backward(s["d_loss"], s["logits"], *teacher, lse, temperature=s["temperature"]))
    if op == "step":
        return dict(o=fl.decay_attention_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"]), state=s["state"])
    qkv, more = (s["q"], s["k"], s["v"], s["log_decay"]), dict(state=s["state"], cu_seqlens=s["cu_seqlens"])
    o, state = fl.decay_attention_forward(*qkv, **more)
    out = dict(o=o, state=state)
    if train:
        out["dq"], out["dk"], out["dv"], out["d_initial"] = fl.decay_attention_backward(s["do"], *qkv, d_state=s["d_state"], **more)
    return out


# ---- the plain forms

def _norm_plain(s):
    x, w, dtype = s["x"].float(), s["weight"], s["x"].dtype
    total = s["x"] if s["residual"] is None else (x + s["residual"].float()).to(dtype)
    t = total.float()
    centred = t - t.mean(-1, keepdim=True)
    rstd = torch.rsqrt((centred * centred).mean(-1, keepdim=True) + 1e-5)
    normed = centred * rstd
    out = dict(y=(normed * w + s["bias"]).to(dtype), total=None if s["residual"] is None else total)
    if s["case"]["call"] == "train":
        dy = s["dy"].float()
        scaled = dy * w
        dx = rstd * (scaled - scaled.mean(-1, keepdim=True) - normed * (scaled * normed).mean(-1, keepdim=True))
        out["dx"] = (dx if s["d_total"] is None else dx + s["d_total"].float()).to(dtype)
        out["dweight"], out["dbias"] = (dy * normed).sum(0), dy.sum(0)
    return out


def _distill_plain(s):
    tau, vocabulary = s["temperature"], s["logits"].shape[1]
    z = s["logits"].float() / tau
    most = z.amax(-1, keepdim=True)
    e = torch.exp(z - most)
    mass = e.sum(-1, keepdim=True)
    lse = most + torch.log(mass)
    index = s["teacher_index"].long()
    held = (index >= 0) & (index < vocabulary)
    index = torch.where(held, index, 0)
    t = torch.where(held, s["teacher_logits"] / tau, -math.inf)
    top = t.amax(-1, keepdim=True)
    any_ = top > -math.inf
    t = torch.where(any_, t - top, -math.inf)
    p = torch.exp(t)
    p = p / torch.where(any_, p.sum(-1, keepdim=True), 1.0)
    log_p = t - torch.log(torch.where(any_, torch.exp(t).sum(-1, keepdim=True), 1.0))
    there = p > 0
    kl = torch.where(there, p * (torch.where(there, log_p, 0.0) - (torch.gather(z, 1, index) - lse)), 0.0).sum(-1)
    out = dict(loss=tau * tau * kl)
    if s["case"]["call"] != "forward":
        d = (tau * s["d_loss"])[:, None]
        grad = e / mass
        grad.scatter_add_(1, index, -p)
        out["dlogits"] = torch.where(any_, d * grad, 0.0).to(s["logits"].dtype)
    return out


def _step_plain(s):
    group = s["case"]["heads"] // s["case"]["kv_heads"]
    q = s["q"].float()
    k, v = (s[name].float().repeat_interleave(group, 1) for name in ("k", "v"))
    state = torch.exp(s["log_decay"])[:, None, None] * s["state"] + k[..., :, None] * v[..., None, :]
    s["state"].copy_(state)
    o = (q[..., :, None] * state).sum(-2) * s["case"]["dk"] ** -0.5
    return dict(o=o.to(s["q"].dtype), state=s["state"])


_CHUNK = 64


def _chunks(x):
    """(N, H, L, D) -> (N, H, L / chunk, chunk, D)."""
    return x.view(*x.shape[:2], -1, _CHUNK, x.shape[-1])


def _attend_plain(s):
    """In chunks of 64 tokens: inside a chunk as masked products, across chunks through the states at their starts, all of which one
    product with the decays between chunks gives."""
    case, lengths = s["case"], s["lengths"]
    heads, group, scale, n, longest = case["heads"], case["heads"] // case["kv_heads"], case["dk"] ** -0.5, len(s["lengths"]), max(s["lengths"])
    dev, padded = s["q"].device, -(-longest // _CHUNK) * _CHUNK
    length = torch.tensor(lengths, device=dev)
    at = torch.arange(padded, device=dev)
    inside = at < length[:, None]                                                  # (N, L)
    row = (length.cumsum(0) - length)[:, None] + at
    row = torch.where(inside, row, 0)

    def spread(x):   # the caller's layout -> (N, heads, L, D) in 32 bits, zeros behind a sequence's end
        x = x.reshape(-1, *x.shape[-2:]).float()[row] * inside[:, :, None, None]
        return x.transpose(1, 2).repeat_interleave(heads // x.shape[2], 1)

    def gather(x, kv=False):   # back, the heads that share keys and values summed
        if kv:
            x = x.view(n, heads // group, group, padded, -1).sum(2)
        return x.transpose(1, 2)[inside].to(s["q"].dtype).view(*s["q"].shape[:-2], x.shape[1], -1)

    q, k, v = spread(s["q"]), spread(s["k"]), spread(s["v"])
    g = s["log_decay"][:, None]                                                    # (H, 1)
    i = torch.arange(_CHUNK, device=dev)
    between = i[:, None] - i
    inner = torch.where(between >= 0, torch.exp(g[..., None] * between.clamp(min=0)), 0.0)[:, None]      # (H, 1, C, C)
    c = torch.arange(padded // _CHUNK, device=dev)
    apart = c[:, None] - c - 1
    across = torch.where(apart >= 0, torch.exp(g[..., None] * (_CHUNK * apart.clamp(min=0))), 0.0)       # (H, nC, nC)
    head, tail = torch.exp(g * (i + 1))[:, None, :, None], torch.exp(g * (_CHUNK - 1 - i))[:, None, :, None]

    def product(a, b):   # sum over a chunk's tokens of a_t b_t
        return a.transpose(-1, -2).contiguous() @ b

    def carried(of_chunks, weights):   # states of all chunks from what each adds
        flat = of_chunks.reshape(*of_chunks.shape[:3], -1)
        return (weights @ flat).view_as(of_chunks)

    def transposed(x):
        return x.transpose(-1, -2).contiguous()

    cq, ck, cv = _chunks(q), _chunks(k), _chunks(v)
    before = carried(product(ck * tail, cv), across) + torch.exp(g * (_CHUNK * c))[:, :, None, None] * s["state"][:, :, None]
    scores = cq @ transposed(ck) * inner
    o = scale * (scores @ cv + head * (cq @ before))
    left = torch.exp(g * (length[:, None, None] - 1 - at).clamp(min=0))[..., None]                       # (N, H, L, 1): decay to the end
    whole = torch.exp(g * length[:, None, None])[..., None]
    state = whole * s["state"] + product(k * left, v)
    out = dict(o=gather(o.view(n, heads, padded, -1)), state=state)
    if case["call"] == "train":
        do = spread(s["do"])
        cdo = _chunks(do)
        pairs = cdo @ transposed(cv) * inner
        dq = scale * (pairs @ ck + head * (cdo @ transposed(before)))
        behind = carried(product(cq * torch.exp(g * i)[:, None, :, None], cdo), transposed(across)) * scale
        reach = torch.exp(g * (_CHUNK - i))[:, None, :, None]
        end = left * inside[:, None, :, None]
        dk = scale * (transposed(pairs) @ cq) + reach * (cv @ transposed(behind))
        dk = dk.view(n, heads, padded, -1) + end * (v @ transposed(s["d_state"]))
        dv = scale * (transposed(scores) @ cdo) + reach * (ck @ behind)
        dv = dv.view(n, heads, padded, -1) + end * (k @ s["d_state"])
        out["dq"], out["dk"], out["dv"] = gather(dq.view(n, heads, padded, -1)), gather(dk, True), gather(dv, True)
        out["d_initial"] = scale * product(q * torch.exp(g * (at + 1))[..., None], do) + whole * s["d_state"]
    return out


def run(s):
    if own:
        return _run_own(s)
    return {"norm": _norm_plain, "distill": _distill_plain, "step": _step_plain, "attend": _attend_plain}[s["case"]["op"]](s)


def work(case):
    """Bytes: every input once, every output once.  Operations: of the norm a few a value; of the loss an exponential and a sum
    a value; of the attention the state's update and use for every token (4 dk dv forward, 12 more backward), which is the least
    that any split into chunks computes."""
    e, op, train = _SIZE[case["dtype"]], case["op"], case["call"] != "forward"
    if op == "norm":
        n, r = case["rows"] * case["width"], case["residual"]
        tensors = (4 if r else 2) + ((3 if r else 2) if train else 0)
        return {"bytes": float(e * n * tensors + 4 * case["width"] * (4 if train else 2)), "flops": 8.0 * n * (2 if train else 1)}
    if op == "distill":
        n = case["rows"] * case["vocabulary"]
        return {"bytes": float(e * n * (2 if train else 1) + case["rows"] * (8 * case["top"] + 8)), "flops": 4.0 * n * (2 if train else 1)}
    n, heads, kv, dk, dv = case["sequences"], case["heads"], case["kv_heads"], case["dk"], case["dv"]
    states = 8 * n * heads * dk * dv
    if op == "step":
        return {"bytes": float(states + e * n * (heads + kv) * (dk + dv)), "flops": 5.0 * n * heads * dk * dv}
    tokens = sum(_lengths(case))
    each = (heads + kv) * (dk + dv)
    if not train:
        return {"bytes": float(states + e * tokens * each), "flops": 4.0 * tokens * heads * dk * dv}
    more = heads * (dk + dv) + kv * (dk + dv)
    return {"bytes": float(2 * states + e * tokens * (each + more)), "flops": 16.0 * tokens * heads * dk * dv}


# ---- the definitions in 64 bits

def _norm_exact(s):
    x = s["x"].double()
    total = x if s["residual"] is None else (x + s["residual"].double()).to(s["x"].dtype).double()   # the stream is held in its type
    variance, mean = torch.var_mean(total, -1, correction=0, keepdim=True)
    normed = (total - mean) / (variance + 1e-5).sqrt()
    out = dict(y=normed * s["weight"].double() + s["bias"].double(), total=None if s["residual"] is None else total)
    if s["case"]["call"] == "train":
        dy, w, width = s["dy"].double(), s["weight"].double(), x.shape[1]
        h = dy * w
        dx = (width * h - h.sum(-1, keepdim=True) - normed * (h * normed).sum(-1, keepdim=True)) / (width * (variance + 1e-5).sqrt())
        out.update(dx=dx if s["d_total"] is None else dx + s["d_total"].double(), dweight=torch.sum(dy * normed, 0), dbias=torch.sum(dy, 0))
    return out


def _distill_exact(s):
    tau, index, vocabulary = s["temperature"], s["teacher_index"].long(), s["logits"].shape[1]
    ignored = (index < 0) | (index >= vocabulary)
    target = torch.softmax((s["teacher_logits"].double() / tau).masked_fill(ignored, -math.inf), -1).nan_to_num(0.0)
    losses, grads = [], []
    for rows in torch.arange(len(index), device=index.device).split(512):   # (a part of the rows at a time: 64 bits of them all are large)
        log_q = torch.log_softmax(s["logits"][rows].double() / tau, -1)
        p = target[rows]
        chosen = log_q.gather(1, index[rows].clamp(0, vocabulary - 1))
        losses.append(tau ** 2 * (torch.special.xlogy(p, p) - p * chosen).sum(-1))
        if s["case"]["call"] != "forward":
            dense = torch.zeros_like(log_q).scatter_add_(1, index[rows].clamp(0, vocabulary - 1), p)
            some = p.sum(-1, keepdim=True) > 0
            grads.append(torch.where(some, s["d_loss"][rows, None].double() * tau * (log_q.exp() - dense), 0.0).float())
    out = dict(loss=torch.cat(losses))
    if grads:
        out["dlogits"] = torch.cat(grads)
    return out


def _step_exact(s):
    group = s["case"]["heads"] // s["case"]["kv_heads"]
    k, v = (s[name].double().repeat_interleave(group, 1) for name in ("k", "v"))
    state = torch.exp(s["log_decay"].double())[None, :, None, None] * s["state"].double() + torch.einsum("nhd,nhe->nhde", k, v)
    return dict(o=torch.einsum("nhd,nhde->nhe", s["q"].double(), state) / math.sqrt(s["case"]["dk"]), state=state)


def _attend_exact(s):
    """The recurrence itself, sequence by sequence and a block of 128 tokens at a time, forward and then back."""
    case, train = s["case"], s["case"]["call"] == "train"
    group, scale, g = case["heads"] // case["kv_heads"], 1 / math.sqrt(case["dk"]), s["log_decay"].double()[:, None, None]

    def heads_first(x, repeat=1):   # (tokens, heads, D) -> (heads, tokens, D)
        return x.double().repeat_interleave(repeat, 1).transpose(0, 1)

    def shared(x):
        return x.view(case["kv_heads"], group, *x.shape[1:]).sum(1)

    names = ["q", "k", "v"] + (["do"] if train else [])
    flat = {name: s[name].reshape(-1, *s[name].shape[-2:]) for name in names}
    parts = {name: [] for name in ("o", "state") + (("dq", "dk", "dv", "d_initial") if train else ())}
    # sequences of one length go together, as more heads
    lengths, starts = s["lengths"], [0]
    for length in lengths:
        starts.append(starts[-1] + length)
    for n, length in enumerate(lengths):
        x = {name: heads_first(flat[name][starts[n]:starts[n + 1]], 1 if name in ("q", "do") else group) for name in names}
        state, kept, outs = s["state"][n].double(), [], []
        for t in range(0, length, 128):
            q, k, v = (x[name][:, t:t + 128] for name in ("q", "k", "v"))
            m = q.shape[1]
            i = torch.arange(m, device=q.device, dtype=torch.float64)
            decay = torch.exp(g * (i[:, None] - i)).tril()
            kept.append((state, decay, i))
            outs.append(scale * (torch.exp(g * (i[:, None] + 1)) * (q @ state) + (decay * (q @ k.mT)) @ v))
            state = torch.exp(g * m) * state + (k * torch.exp(g * (m - 1 - i[:, None]))).mT @ v
        parts["o"].append(torch.cat(outs, 1).transpose(0, 1))
        parts["state"].append(state)
        if not train:
            continue
        grad, back = s["d_state"][n].double(), []          # the gradient of the state behind the block
        for block in reversed(range(len(kept))):
            state, decay, i = kept[block]
            q, k, v, do = (x[name][:, block * 128:block * 128 + 128] for name in names)
            m = q.shape[1]
            early, late = torch.exp(g * (i[:, None] + 1)), torch.exp(g * (m - 1 - i[:, None]))
            of_scores = scale * decay * (do @ v.mT)
            dq = of_scores @ k + scale * early * (do @ state.mT)
            dk = of_scores.mT @ q + late * (v @ grad.mT)
            dv = scale * (decay * (q @ k.mT)).mT @ do + late * (k @ grad)
            grad = torch.exp(g * m) * grad + scale * (q * early).mT @ do
            back.append((dq, shared(dk), shared(dv)))
        for name, pieces in zip(("dq", "dk", "dv"), zip(*reversed(back))):
            parts[name].append(torch.cat(pieces, 1).transpose(0, 1))
        parts["d_initial"].append(grad)
    out = {}
    for name, pieces in parts.items():
        whole = torch.stack(pieces) if name in ("state", "d_initial") else torch.cat(pieces)
        like = {"o": "q", "dq": "q", "dk": "k", "dv": "v"}.get(name)
        out[name] = whole if like is None else whole.reshape(*s[like].shape[:-1], whole.shape[-1])
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _norm_exact, "distill": _distill_exact, "step": _step_exact, "attend": _attend_exact}[case["op"]](s)
