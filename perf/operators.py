"""Workloads of the causal-transformer operators beside transformer.py's encoder attention: rotary positions, attention
over packed sequences of different lengths (causal, grouped heads, with its gradient), rotary positions written into a
paged key/value cache, and attention of new tokens over that cache.

Every operator has a plain form here (elementary torch operations, 32-bit arithmetic, 64-bit angles) and a call of the
framework's entry point, chosen by `own`.  Shapes: q [tokens, heads, dim], k and v [tokens, kv heads, dim], query head h
reading kv head h // (heads / kv heads); pages [pages, page size, kv heads, dim]."""
import math
import random

import numpy as np
import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}


def _text(lengths):
    return " ".join(map(str, lengths))      # a case holds its lengths as text


def _ints(case, name):
    return [int(x) for x in case[name].split()]


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # rotary positions of one training batch at the critic's headline shape (64 sequences of 512 calls, 4 heads of 16),
        # forward and backward, pairs side by side
        dict(name="rotary_train_fp32", op="rotary", type="fp32", tokens=64 * 512, heads=4, kv_heads=4, dim=16, rotary=16,
             interleaved=True, backward=True, first=0, factor=1.0, base=10000.0),
        # the rotation before attention over a long prompt, grouped heads, halves
        dict(name="rotary_prompt_bf16", op="rotary", type="bf16", tokens=16383, heads=32, kv_heads=8, dim=128, rotary=128,
             interleaved=False, backward=False, first=0, factor=1.0, base=10000.0),
        # one decoding step of 48 sequences far into a stretched context: half of each head is rotated
        dict(name="append_step_fp16", op="append", type="fp16", new=_text([1] * 48), context=_text(30011 + 997 * (i % 7) for i in range(48)),
             heads=12, kv_heads=4, dim=96, rotary=48, interleaved=True, page=16, factor=8.0, base=10000.0),
        # a chunk of prompts entering the cache
        dict(name="append_prompt_bf16", op="append", type="bf16", new="2047 900 1501 3", context="2047 1000 5000 777",
             heads=32, kv_heads=8, dim=128, rotary=128, interleaved=False, page=64, factor=1.0, base=500000.0),
        # training on ragged traces at the framework's own attention shape: 64 sequences of at most 512, 4 heads of 16, fp32
        dict(name="packed_train_fp32", op="packed", type="fp32", lengths=_text(512 - (i * 37) % 449 for i in range(64)),
             heads=4, kv_heads=4, dim=16, backward=True),
        # many short sequences with odd lengths, one kv head for all query heads
        dict(name="packed_train_short_fp16", op="packed", type="fp16", lengths=_text(1 + (i * 53) % 203 for i in range(96)),
             heads=12, kv_heads=1, dim=64, backward=True),
        # training on long packed sequences
        dict(name="packed_train_bf16", op="packed", type="bf16", lengths="4096 2049 1000 4001 333 2800 64 2041",
             heads=16, kv_heads=4, dim=128, backward=True),
        # prompts processed together before decoding
        dict(name="packed_prompt_bf16", op="packed", type="bf16", lengths="8191 1025 5000", heads=32, kv_heads=8, dim=128,
             backward=False),
        # one sequence, one token, short context: latency
        dict(name="paged_one_fp32", op="paged", type="fp32", new="1", context="777", heads=8, kv_heads=2, dim=64, page=16),
        # one decoding step of a batch with mixed contexts
        dict(name="paged_step_bf16", op="paged", type="bf16", new=_text([1] * 64), context=_text(300 + (i * 1237) % 7893 for i in range(64)),
             heads=32, kv_heads=8, dim=128, page=16),
        # one decoding step of two very long contexts
        dict(name="paged_long_fp16", op="paged", type="fp16", new="1 1", context="131071 90001", heads=16, kv_heads=2,
             dim=96, page=64),
        # chunks of new tokens over what the cache holds already, one of them a short continuation
        dict(name="paged_chunk_bf16", op="paged", type="bf16", new="512 301 777 5", context="9000 301 16001 4000",
             heads=32, kv_heads=8, dim=128, page=32),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng: random.Random):
    op = rng.choice(["rotary", "append", "packed", "packed", "paged", "paged"])
    typ = rng.choice(["fp32", "bf16", "fp16"])
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 2, 3, 4, 8] if kv < 8 else [1, 2, 4])
    dim = rng.choice([16, 32, 48, 64, 80, 96, 128])
    rotary = rng.choice([dim, dim, dim // 2])
    turn = dict(rotary=rotary, interleaved=rng.random() < 0.5, factor=rng.choice([1.0, 4.0, 8.0]), base=rng.choice([10000.0, 500000.0]))
    case = dict(op=op, type=typ, heads=heads, kv_heads=kv, dim=dim)
    if op == "rotary":
        return case | turn | dict(tokens=_log_int(rng, 1, 16000), backward=rng.random() < 0.5, first=rng.choice([0, _log_int(rng, 1, 1000000)]))
    if op == "packed":
        # the widest score matrix, padded: at most 64 x 2^20 of them
        longest = _log_int(rng, 1, 4500)
        most = max(1, min(128, 30000 // longest, (64 << 20) // (heads * longest * longest)))
        n = _log_int(rng, 1, most)
        lengths = [longest] + [_log_int(rng, 1, longest) for _ in range(n - 1)]
        rng.shuffle(lengths)
        return case | dict(lengths=_text(lengths), backward=rng.random() < 0.6)
    page = rng.choice([16, 32, 64, 128])
    longest = _log_int(rng, 1, 60000)
    n = _log_int(rng, 1, max(1, min(96, 200000 // longest)))
    context = [longest] + [_log_int(rng, 1, longest) for _ in range(n - 1)]
    rng.shuffle(context)
    single = rng.random() < 0.5
    chunk = max(1, (32 << 20) // (heads * longest * n))
    new = [1 if single else _log_int(rng, 1, min(c, 1500, chunk)) for c in context]
    return case | (turn if op == "append" else {}) | dict(new=_text(new), context=_text(context), page=page)


# ---------------------------------------------------------------------------------------------------------------- inputs
def _starts(lengths):
    return [0] + np.cumsum(lengths).tolist()


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    dt, op = TYPES[case["type"]], case["op"]
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    rows = case["tokens"] if op == "rotary" else sum(_ints(case, "lengths")) if op == "packed" else sum(_ints(case, "new"))
    # q, k and v are the three parts of one projection, as a model has them
    qkv = torch.randn(rows, (H + 2 * Hk) * D, generator=g, device=dev).to(dt)
    s = dict(case=case, q=qkv[:, :H * D].view(rows, H, D), k=qkv[:, H * D:(H + Hk) * D].view(rows, Hk, D),
             v=qkv[:, (H + Hk) * D:].view(rows, Hk, D), scale=1.0 / math.sqrt(D), handle=None)
    if op in ("rotary", "append"):
        R = case["rotary"]
        # radians per position of each pair; a longer context is reached by a slower turn
        s["frequencies"] = (case["base"] ** (-torch.arange(0, R, 2, dtype=torch.float64) / R) / case["factor"]).to(dev)
        s["multiplier"] = 1.0 + 0.1 * math.log(case["factor"])
    if case.get("backward"):
        s["grads"] = [torch.randn(rows, H, D, generator=g, device=dev).to(dt)]
        if op == "rotary":
            s["grads"].append(torch.randn(rows, Hk, D, generator=g, device=dev).to(dt))
    if op == "rotary":
        s["positions"] = torch.arange(rows, device=dev, dtype=torch.int32) % 8192 + case["first"]
    if op == "packed":
        lengths = _ints(case, "lengths")
        s["starts"] = torch.tensor(_starts(lengths), device=dev)
        s["lengths"], s["longest"] = torch.tensor(lengths, device=dev), max(lengths)
    if op in ("append", "paged"):
        page, n = case["page"], len(_ints(case, "new"))
        need = [-(-c // page) for c in _ints(case, "context")]
        pages = sum(need) + 3
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
        table = torch.zeros(n, max(need), dtype=torch.int32)
        for i, m in enumerate(need):
            table[i, :m] = torch.tensor(order[:m], dtype=torch.int32)
            order = order[m:]
        s["table"] = table.to(dev)
        s["context"] = torch.tensor(_ints(case, "context"), device=dev, dtype=torch.int32)
        s["starts"] = torch.tensor(_starts(_ints(case, "new")), device=dev)
        s["lengths"], s["longest"] = torch.tensor(_ints(case, "new"), device=dev), max(_ints(case, "new"))
        s["keys"] = torch.randn(pages, page, Hk, D, generator=g, device=dev).to(dt)
        s["values"] = torch.randn(pages, page, Hk, D, generator=g, device=dev).to(dt)
    if own:
        import transformer
        # what a program keeps for a batch: its layout, made from the lengths it knows on the host
        if op == "packed":
            s["handle"] = transformer.PackedSequences(_ints(case, "lengths"), dev)
        if op in ("append", "paged"):
            s["handle"] = transformer.PagedBatch(s["table"], _ints(case, "context"), _ints(case, "new"))
    return s


# ----------------------------------------------------------------------------------------------------- plain forms, calls
def _turned(x, cos, sin, rotary, interleaved, multiplier, back=False):
    """The first `rotary` features of every head turned by the angles [rows, rotary / 2] (the other way round for gradients)."""
    y = x.float()
    a, b = (y[..., 0:rotary:2], y[..., 1:rotary:2]) if interleaved else (y[..., :rotary // 2], y[..., rotary // 2:rotary])
    c, s = cos[:, None] * multiplier, sin[:, None] * (-multiplier if back else multiplier)
    u, w = a * c - b * s, a * s + b * c
    turned = torch.stack((u, w), -1).flatten(-2) if interleaved else torch.cat((u, w), -1)
    return torch.cat((turned, y[..., rotary:]), -1).to(x.dtype)


def _cos_sin(positions, frequencies):
    angles = positions.double()[:, None] * frequencies
    return angles.cos().float(), angles.sin().float()


def _plain_rotary(s):
    c = s["case"]
    cos, sin = _cos_sin(s["positions"], s["frequencies"])
    turn = (cos, sin, c["rotary"], c["interleaved"], s["multiplier"])
    out = [_turned(s["q"], *turn), _turned(s["k"], *turn)]
    return out + [_turned(g, *turn, back=True) for g in s.get("grads", [])]


def _padded(x, starts, lengths, longest):
    at = torch.arange(longest, device=x.device)
    valid = at < lengths[:, None]
    return x.float()[(starts[:-1, None] + at).clamp(max=x.shape[0] - 1)], valid


def _plain_attention(q, k, v, allowed, scale, do=None):
    """q [n, L, H, D], k and v [n, M, Hk, D] in 32 bits, allowed [n, L, M]; rows with no key give zeros."""
    n, L, H, D = q.shape
    M, Hk = k.shape[1:3]
    group = lambda x: x.view(n, L, Hk, H // Hk, D).permute(0, 2, 3, 1, 4).reshape(n, Hk, H // Hk * L, D)  # noqa: E731
    back = lambda x: x.view(n, Hk, H // Hk, L, D).permute(0, 3, 1, 2, 4).reshape(n, L, H, D)  # noqa: E731
    q, k, v = group(q), k.transpose(1, 2).contiguous(), v.transpose(1, 2).contiguous()
    p = q @ k.transpose(2, 3)
    p = p.mul_(scale).view(n, Hk, H // Hk, L, M).masked_fill_(~allowed[:, None, None], -math.inf)
    p = p.sub_(p.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    p = p.div_(p.sum(-1, keepdim=True).clamp(min=1e-30)).view(n, Hk, H // Hk * L, M)
    if do is None:
        return back(p @ v)
    do = group(do)
    dp = do @ v.transpose(2, 3)
    dp = dp.sub_((dp * p).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    return back(p @ v), back(dp @ k), (dp.transpose(2, 3) @ q).transpose(1, 2), (p.transpose(2, 3) @ do).transpose(1, 2)


def _rows(s):
    """(sequence, row in it) of every packed row."""
    n, rows = s["lengths"].shape[0], s["q"].shape[0]
    seq = torch.repeat_interleave(torch.arange(n, device=s["q"].device), s["lengths"], output_size=rows)
    return seq, torch.arange(rows, device=seq.device) - s["starts"][seq]


def _plain_packed(s):
    L = s["longest"]
    q, valid = _padded(s["q"], s["starts"], s["lengths"], L)
    k, v = (_padded(s[x], s["starts"], s["lengths"], L)[0] for x in "kv")
    at = torch.arange(L, device=q.device)
    allowed = (at[None, :] <= at[:, None]) & valid[:, None, :]
    if not s["case"]["backward"]:
        return [_plain_attention(q, k, v, allowed, s["scale"])[_rows(s)].to(s["q"].dtype)]
    do = _padded(s["grads"][0], s["starts"], s["lengths"], L)[0] * valid[..., None, None]
    return [x[_rows(s)].to(s["q"].dtype) for x in _plain_attention(q, k, v, allowed, s["scale"], do)]


def _plain_append(s):
    c = s["case"]
    seq, at = _rows(s)
    at = at + (s["context"].long() - s["lengths"])[seq]      # the new tokens are the last of their sequences
    turn = (*_cos_sin(at, s["frequencies"]), c["rotary"], c["interleaved"], s["multiplier"])
    where = (s["table"].long()[seq, at // c["page"]], at % c["page"])
    s["keys"][where] = _turned(s["k"], *turn)
    s["values"][where] = s["v"]
    return [_turned(s["q"], *turn), s["keys"], s["values"]]


def _plain_paged(s):
    n, Hk, D = s["lengths"].shape[0], s["case"]["kv_heads"], s["case"]["dim"]
    q, _ = _padded(s["q"], s["starts"], s["lengths"], s["longest"])
    k, v = (s[x][s["table"].long()].view(n, -1, Hk, D).float() for x in ("keys", "values"))
    at, row = torch.arange(k.shape[1], device=k.device), torch.arange(q.shape[1], device=k.device)
    last = (s["context"].long() - s["lengths"])[:, None] + row
    return [_plain_attention(q, k, v, (at <= last[..., None]) & (at < s["context"][:, None, None]), s["scale"])[_rows(s)].to(s["q"].dtype)]


def _own_rotary(s):
    import transformer
    c = s["case"]
    how = dict(interleaved=c["interleaved"], multiplier=s["multiplier"])
    if not c["backward"]:
        return list(transformer.apply_rotary(s["q"], s["k"], s["positions"], s["frequencies"], **how))
    q, k = s["q"].detach().requires_grad_(), s["k"].detach().requires_grad_()
    out = transformer.apply_rotary(q, k, s["positions"], s["frequencies"], **how)
    return [*(x.detach() for x in out), *torch.autograd.grad(out, (q, k), s["grads"])]


def _own_packed(s):
    import transformer
    if not s["case"]["backward"]:
        return [transformer.packed_attention(s["q"], s["k"], s["v"], s["handle"], scale=s["scale"])]
    q, k, v = (s[x].detach().requires_grad_() for x in "qkv")
    out = transformer.packed_attention(q, k, v, s["handle"], scale=s["scale"])
    return [out.detach(), *torch.autograd.grad(out, (q, k, v), s["grads"][0])]


def _own_append(s):
    import transformer
    c = s["case"]
    q = transformer.append_rotary(s["q"], s["k"], s["v"], s["keys"], s["values"], s["handle"], s["frequencies"],
                                  interleaved=c["interleaved"], multiplier=s["multiplier"])
    return [q, s["keys"], s["values"]]


def _own_paged(s):
    import transformer
    return [transformer.paged_attention(s["q"], s["keys"], s["values"], s["handle"], scale=s["scale"])]


def run(state):
    forms = (dict(rotary=_own_rotary, packed=_own_packed, append=_own_append, paged=_own_paged) if own else
             dict(rotary=_plain_rotary, packed=_plain_packed, append=_plain_append, paged=_plain_paged))
    return forms[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------------------------------ work
def work(case):
    b, H, Hk, D, op = BYTES[case["type"]], case["heads"], case["kv_heads"], case["dim"], case["op"]
    if op == "rotary":
        # every element read once and written once; a turned pair takes 4 products and 2 sums
        rows, ways = case["tokens"], 2 if case["backward"] else 1
        return {"bytes": ways * 2 * rows * (H + Hk) * D * b + 4 * rows, "flops": ways * 3 * rows * (H + Hk) * case["rotary"]}
    if op == "append":
        rows = sum(_ints(case, "new"))
        return {"bytes": 2 * rows * (H + 2 * Hk) * D * b, "flops": 3 * rows * (H + Hk) * case["rotary"]}
    if op == "packed":
        rows, pairs = sum(_ints(case, "lengths")), sum(n * (n + 1) // 2 for n in _ints(case, "lengths"))
        # two products forward; backward five, the scores among them (no matrix of scores is kept)
        if not case["backward"]:
            return {"bytes": rows * (2 * H + 2 * Hk) * D * b, "flops": 4 * pairs * H * D}
        return {"bytes": rows * (4 * H + 4 * Hk) * D * b, "flops": 14 * pairs * H * D}
    pairs = sum(n * c - n * (n - 1) // 2 for n, c in zip(_ints(case, "new"), _ints(case, "context")))
    return {"bytes": (2 * sum(_ints(case, "new")) * H + 2 * sum(_ints(case, "context")) * Hk) * D * b, "flops": 4 * pairs * H * D}


# --------------------------------------------------------------------------------------- the definitions, in 64 bits
def _exact_turn(x, angles, case, multiplier, sign=1.0):
    """The pairs as complex numbers times multiplier * exp(i sign angle)."""
    R = case["rotary"]
    y = x.double().clone()
    low = torch.arange(R // 2, device=x.device)
    first, second = (2 * low, 2 * low + 1) if case["interleaved"] else (low, low + R // 2)
    z = torch.complex(y[..., first], y[..., second]) * torch.polar(torch.full_like(angles, multiplier), sign * angles)[:, None]
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_head(q, k, v, first, scale, do=None):
    """One head of one sequence: row i sees keys 0 .. first + i.  The weights are exp(score - log of the row's sum)."""
    score = (q @ k.T) * scale
    hidden = torch.arange(k.shape[0], device=q.device)[None, :] > (first + torch.arange(q.shape[0], device=q.device))[:, None]
    score[hidden] = -math.inf
    weight = torch.exp(score - torch.logsumexp(score, 1, keepdim=True))
    out = weight @ v
    if do is None:
        return out
    # d score = weight (dO . v - dO . out)
    ds = weight * (do @ v.T - (do * out).sum(1, keepdim=True)) * scale
    return out, ds @ k, ds.T @ q, weight.T @ do


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    H, Hk = case["heads"], case["kv_heads"]
    q, k, v = (s[x].double() for x in "qkv")
    G = H // Hk
    if op == "rotary":
        angles = torch.outer(s["positions"].double(), s["frequencies"])
        return [_exact_turn(s["q"], angles, case, s["multiplier"]), _exact_turn(s["k"], angles, case, s["multiplier"]),
                *(_exact_turn(g, angles, case, s["multiplier"], -1.0) for g in s.get("grads", []))]
    if op == "packed":
        out = [torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)]
        row = 0
        for n in _ints(case, "lengths"):
            at = slice(row, row + n)
            for h in range(H):
                j = h // G
                if case["backward"]:
                    o, dq, dk, dv = _exact_head(q[at, h], k[at, j], v[at, j], 0, s["scale"], s["grads"][0][at, h].double())
                    out[1][at, h] = dq
                    out[2][at, j] += dk
                    out[3][at, j] += dv
                else:
                    o = _exact_head(q[at, h], k[at, j], v[at, j], 0, s["scale"])
                out[0][at, h] = o
            row += n
        return out if case["backward"] else out[:1]
    table, page, row = s["table"].cpu().long(), case["page"], 0
    if op == "append":
        keys, values, turned, row = s["keys"].double(), s["values"].double(), torch.zeros_like(q), 0
        for i, (n, c) in enumerate(zip(_ints(case, "new"), _ints(case, "context"))):
            at, where = slice(row, row + n), np.arange(c - n, c)
            angles = torch.outer(torch.from_numpy(where).to(q.device).double(), s["frequencies"])
            turned[at] = _exact_turn(s["q"][at], angles, case, s["multiplier"])
            index = (table[i][where // page].to(q.device), torch.from_numpy(where % page).to(q.device))
            keys[index] = _exact_turn(s["k"][at], angles, case, s["multiplier"])
            values[index] = v[at]
            row += n
        return [turned, keys, values]
    out = torch.zeros_like(q)
    for i, (n, c) in enumerate(zip(_ints(case, "new"), _ints(case, "context"))):
        mine = table[i, :-(-c // page)].to(q.device)
        k, v = (s[x][mine].flatten(0, 1)[:c].double() for x in ("keys", "values"))
        for h in range(H):
            out[row:row + n, h] = _exact_head(q[row:row + n, h], k[:, h // G], v[:, h // G], c - n, s["scale"])
        row += n
    return [out]
