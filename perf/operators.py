"""Cases of the serving operators: rotary positions, attention over a shared prefix, rules on logits.

``run`` computes each operator in its plain form (elementary torch operations in 32 bits), or, with ``own``
set, through the framework's own entry points.  ``exact`` is the definition in 64 bits.
"""

import math

import torch

own = False

F32 = torch.float32
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
HEADS = [(32, 8), (28, 4), (12, 12), (8, 2), (32, 4)]  # query heads, key/value heads


# ---------------------------------------------------------------------------------- cases

def listed():
    return [
        # one decode step of 64 requests far into their contexts: the smallest call, latency counts
        dict(name="rotary step", op="rotary", tokens=64, heads=32, kv_heads=8, dim=128, rot=128, layout="half",
             dtype="bf16", grad=False, max_pos=131072, factor=8.0),
        # a training batch of 8 x 1,024 tokens, interleaved pairs over half of the head, with gradients
        dict(name="rotary train", op="rotary", tokens=8192, heads=32, kv_heads=8, dim=128, rot=64,
             layout="interleaved", dtype="bf16", grad=True, max_pos=1024, factor=1.0),
        # prefill of 4 prompts of 4,096 tokens straight from the fused projection into the cache rows
        dict(name="rotary prefill cache", op="rotary_cache", tokens=16384, heads=32, kv_heads=8, dim=128, rot=128,
             layout="half", dtype="bf16", max_pos=8192, factor=4.0, padded=0.1),
        # few requests behind a short system prompt: latency counts
        dict(name="prefix decode small", op="prefix", batch=8, tokens=1, prefix=2048, lo=16, hi=128, cap=160, heads=32,
             kv_heads=8, dim=128, ragged=False),
        # the ordinary decode batch: 64 requests behind an 8K prompt, own parts of 64 to 1,024 tokens
        dict(name="prefix decode", op="prefix", batch=64, tokens=1, prefix=8192, lo=64, hi=1024, cap=1280, heads=32,
             kv_heads=8, dim=128, ragged=False),
        # a large decode batch behind a 32K document, 7 query heads to a key/value head
        dict(name="prefix decode large", op="prefix", batch=128, tokens=1, prefix=32768, lo=128, hi=2048, cap=2048,
             heads=28, kv_heads=4, dim=128, ragged=False),
        # drafted tokens checked five at a time, head dim 64, odd prefix, rows that share different parts of it
        dict(name="prefix drafts", op="prefix", batch=16, tokens=5, prefix=4099, lo=5, hi=300, cap=333, heads=12,
             kv_heads=12, dim=64, ragged=True),
        # prefill of the requests' own 512 tokens behind a 16K prompt: bound by the products
        dict(name="prefix suffix prefill", op="prefix", batch=4, tokens=512, prefix=16384, lo=512, hi=512, cap=640,
             heads=32, kv_heads=8, dim=128, ragged=False),
        # the greedy token of one request under a grammar: the smallest call
        dict(name="choose one", op="choose", batch=1, vocab=128256, dtype="bf16", history=512, biases=16, mask=True),
        # the greedy tokens of a large batch with long histories
        dict(name="choose batch", op="choose", batch=256, vocab=152064, dtype="bf16", history=8192, biases=0, mask=True),
        # every rule on the logits of a decode batch, written back for a sampler
        dict(name="process batch", op="process", batch=64, vocab=128256, dtype="bf16", history=1024, biases=64, mask=True),
        # odd vocabulary in 32 bits, penalties only
        dict(name="process fp32 odd", op="process", batch=33, vocab=50257, dtype="fp32", history=300, biases=0, mask=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    op = rng.choice(["rotary", "rotary_cache", "prefix", "prefix", "prefix", "choose", "process"])
    heads, kv = rng.choice(HEADS)
    dim = rng.choice([64, 128])
    if op in ("rotary", "rotary_cache"):
        case = dict(op=op, tokens=_log(rng, 1, 16384), heads=heads, kv_heads=kv, dim=dim,
                    rot=rng.choice([dim, dim, dim // 2, dim // 4 + 2 * rng.randint(0, 3)]),
                    layout=rng.choice(["half", "interleaved"]),
                    dtype="bf16" if op == "rotary_cache" else rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                    max_pos=_log(rng, 16, 131072), factor=rng.choice([1.0, 2.0, 8.0]))
        if op == "rotary":
            case["grad"] = rng.random() < 0.4
        else:
            case["padded"] = rng.choice([0.0, 0.2])
        return case
    if op == "prefix":
        tokens = rng.choice([1, 1, 1, rng.randint(2, 9), _log(rng, 10, 512)])
        hi = tokens + _log(rng, 1, 1500)
        return dict(op=op, batch=_log(rng, 1, 128), tokens=tokens, prefix=_log(rng, 1, 32768), lo=tokens, hi=hi,
                    cap=hi + rng.randint(0, 40), heads=heads, kv_heads=kv, dim=dim, ragged=rng.random() < 0.3)
    return dict(op=op, batch=_log(rng, 1, 256), vocab=rng.choice([32768, 50257, 128256, 152064, _log(rng, 100, 150000)]),
                dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), history=rng.choice([0, _log(rng, 1, 16384)]),
                biases=rng.choice([0, _log(rng, 1, 300)]), mask=rng.random() < 0.6)


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        kind = "rotary" if c["op"].startswith("rotary") else "prefix" if c["op"] == "prefix" else "logits"
        best = most.get(kind, (0, 0))
        most[kind] = (max(best[0], w["bytes"]), max(best[1], w["flops"]))
    while True:
        case = _draw(rng)
        kind = "rotary" if case["op"].startswith("rotary") else "prefix" if case["op"] == "prefix" else "logits"
        w = work(case)
        if w["bytes"] <= most[kind][0] and w["flops"] <= most[kind][1]:
            return case


def _lengths(case):
    """Own lengths of the rows: spread evenly over lo .. hi (the seed only deals them out)."""
    b, lo, hi = case["batch"], case["lo"], case["hi"]
    return [hi if b == 1 else lo + (hi - lo) * i // (b - 1) for i in range(b)]


def _prefix_lengths(case):
    b, p = case["batch"], case["prefix"]
    return [p if not case["ragged"] else p * ((i * 7) % (b + 1)) // b for i in range(b)]


def work(case):
    op = case["op"]
    if op in ("rotary", "rotary_cache"):
        size = DTYPES[case["dtype"]].itemsize
        n, h, kv, d, rot = (case[k] for k in ("tokens", "heads", "kv_heads", "dim", "rot"))
        table = min(n, case["max_pos"]) * rot * 4  # cos and sin rows of the positions met
        if op == "rotary_cache":
            return {"bytes": 2 * n * (h + 2 * kv) * d * size + table + 12 * n, "flops": 3 * n * (h + kv) * rot}
        passes = 2 if case["grad"] else 1
        return {"bytes": passes * 2 * n * (h + kv) * d * size + table + 4 * n, "flops": passes * 3 * n * (h + kv) * rot}
    if op == "prefix":
        b, t, h, kv, d = (case[k] for k in ("batch", "tokens", "heads", "kv_heads", "dim"))
        lens, pre = _lengths(case), _prefix_lengths(case)
        pairs = sum(t * p + t * n - t * (t - 1) // 2 for n, p in zip(lens, pre))
        return {"bytes": 4 * kv * d * (max(pre) + sum(lens)) + 4 * b * t * h * d + 4 * b * t * h, "flops": 4 * h * d * pairs}
    b, v = case["batch"], case["vocab"]
    size = DTYPES[case["dtype"]].itemsize
    read = b * v * size + 4 * b * case["history"] + 8 * b * case["biases"] + (b * v // 8 if case["mask"] else 0)
    return {"bytes": read + (b * v * size if op == "process" else 12 * b), "flops": 4 * b * v}


# ---------------------------------------------------------------------------------- inputs

def _tables(case, device):
    """cos / sin ``[max_pos, rot / 2]``, angles in 64 bits; positions divided by ``factor``."""
    half = case["rot"] // 2
    inv = 500000.0 ** (-torch.arange(half, dtype=torch.float64, device=device) / half) / case["factor"]
    angle = torch.arange(case["max_pos"], dtype=torch.float64, device=device)[:, None] * inv
    return angle.cos().float(), angle.sin().float()


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)

    def randn(*shape, dtype=torch.bfloat16, scale=1.0):
        return (torch.randn(*shape, generator=gen, device=dev) * scale).to(dtype)

    def randint(lo, hi, shape, dtype=torch.int32):
        return torch.randint(lo, hi, shape, generator=gen, device=dev).to(dtype)

    op, s = case["op"], {"case": case}
    if op in ("rotary", "rotary_cache"):
        n, h, kv, d = (case[k] for k in ("tokens", "heads", "kv_heads", "dim"))
        dtype = DTYPES[case["dtype"]]
        s["cos"], s["sin"] = _tables(case, dev)
        s["positions"] = randint(0, case["max_pos"], (n,))
        if op == "rotary":
            s["q"], s["k"] = randn(n, h, d, dtype=dtype), randn(n, kv, d, dtype=dtype)
            if case["grad"]:
                s["q"].requires_grad_()
                s["k"].requires_grad_()
                s["dq"], s["dk"] = randn(n, h, d, dtype=dtype), randn(n, kv, d, dtype=dtype)
        else:
            s["qkv"] = randn(n, (h + 2 * kv) * d, dtype=dtype)
            slots = torch.randperm(n + 64, generator=gen, device=dev)[:n].to(torch.int32)
            s["slots"] = torch.where(torch.rand(n, generator=gen, device=dev) < case["padded"], -1, slots).to(torch.int32)
            s["k_cache"], s["v_cache"] = randn(n + 64, kv * d, dtype=dtype), randn(n + 64, kv * d, dtype=dtype)
        return s
    if op == "prefix":
        b, t, h, kv, d, p = (case[k] for k in ("batch", "tokens", "heads", "kv_heads", "dim", "prefix"))
        s["q"] = randn(b, t, h * d, scale=1.5)
        s["pk"], s["pv"] = randn(p, kv * d), randn(p, kv * d)
        s["k"], s["v"] = randn(b, case["cap"], kv * d), randn(b, case["cap"], kv * d)
        deal = torch.randperm(b, generator=gen, device=dev)
        s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device=dev)[deal]
        s["prefix_lengths"] = torch.tensor(_prefix_lengths(case), dtype=torch.int32, device=dev)[deal] if case["ragged"] else None
        return s
    b, v = case["batch"], case["vocab"]
    s["logits"] = randn(b, v, dtype=DTYPES[case["dtype"]], scale=2.5)
    s["repetition"] = 1.0 + 0.5 * torch.rand(b, generator=gen, device=dev)
    s["presence"] = torch.rand(b, generator=gen, device=dev)
    s["frequency"] = 0.3 * torch.rand(b, generator=gen, device=dev)
    n = case["history"]
    if n:
        # ids crowd towards the front of the vocabulary, as words do
        s["ids"] = (v * torch.rand(b, n, generator=gen, device=dev) ** 4).to(torch.int32).clamp_(max=v - 1)
        s["hist_len"] = torch.full((b,), n, dtype=torch.int32, device=dev)
        s["prompt_len"] = randint(0, n + 1, (b,))
    else:
        s["ids"] = s["hist_len"] = s["prompt_len"] = None
    if case["biases"]:
        s["bias_ids"] = torch.stack([torch.randperm(v, generator=gen, device=dev)[: min(v, case["biases"])] for _ in range(b)]).to(torch.int32)
        s["bias_values"] = randn(*s["bias_ids"].shape, dtype=F32, scale=3.0)
    else:
        s["bias_ids"] = s["bias_values"] = None
    s["mask"] = randint(-2 ** 31, 2 ** 31, (b, (v + 31) // 32), dtype=torch.int32) if case["mask"] else None
    return s


# ---------------------------------------------------------------------------------- plain forms

def _rotate(x, cos, sin, rot, interleaved):
    """``x`` ``[N, H, D]`` in 32 bits, cos / sin ``[N, rot / 2]``."""
    c, s = cos[:, None, :], sin[:, None, :]
    y = x.clone()
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., : rot // 2], x[..., rot // 2: rot]
        y[..., : rot // 2], y[..., rot // 2: rot] = a * c - b * s, b * c + a * s
    return y


def _plain_rotary(s):
    case = s["case"]
    pos = s["positions"].long()
    cos, sin, inter = s["cos"][pos], s["sin"][pos], case["layout"] == "interleaved"
    if case["op"] == "rotary":
        with torch.no_grad():
            out = [_rotate(s[n].float(), cos, sin, case["rot"], inter).to(s[n].dtype) for n in ("q", "k")]
            if case["grad"]:
                out += [_rotate(s[n].float(), cos, -sin, case["rot"], inter).to(s[n].dtype) for n in ("dq", "dk")]
        return out
    n, h, kv, d = (case[k] for k in ("tokens", "heads", "kv_heads", "dim"))
    x = s["qkv"].float().view(n, h + 2 * kv, d)
    qk = _rotate(x[:, : h + kv], cos, sin, case["rot"], inter)
    # the token of each cache row, -1 where none of the batch writes it (padded tokens have slot -1)
    rows = s["k_cache"].shape[0]
    place = torch.where(s["slots"] >= 0, s["slots"], rows).long()
    token = torch.full((rows + 1,), -1, device=place.device).scatter(0, place, torch.arange(n, device=place.device))[:rows]
    written, token = (token >= 0)[:, None], token.clamp(min=0)
    s["k_cache"].copy_(torch.where(written, qk[token, h:].reshape(rows, kv * d).to(s["k_cache"].dtype), s["k_cache"]))
    s["v_cache"].copy_(torch.where(written, x[token, h + kv:].reshape(rows, kv * d).to(s["v_cache"].dtype), s["v_cache"]))
    return qk[:, :h].reshape(n, h * d).to(s["qkv"].dtype), s["k_cache"], s["v_cache"]


def _plain_prefix(s):
    case = s["case"]
    b, t, h, kv, d, p, cap = (case[k] for k in ("batch", "tokens", "heads", "kv_heads", "dim", "prefix", "cap"))
    g = h // kv
    neg = float("-inf")
    q = (s["q"].float() / math.sqrt(d)).view(b, t, kv, g, d).permute(2, 0, 1, 3, 4).reshape(kv, b * t * g, d)
    pk, pv = s["pk"].float().view(p, kv, d), s["pv"].float().view(p, kv, d)
    lk, lv = s["k"].float().view(b, cap, kv, d), s["v"].float().view(b, cap, kv, d)
    sp = torch.matmul(q, pk.permute(1, 2, 0))                                          # [kv, b t g, p]
    ql = q.view(kv, b, t * g, d)
    sl = torch.matmul(ql, lk.permute(2, 0, 3, 1)).view(kv, b, t, g, cap)               # [kv, b, t, g, cap]
    if s["prefix_lengths"] is not None:
        seen = torch.arange(p, device=q.device) < s["prefix_lengths"][:, None]
        sp.view(kv, b, t * g, p).masked_fill_(~seen[None, :, None], neg)
    last = s["lengths"][:, None] - t + torch.arange(t, device=q.device)                # [b, t] last visible own key
    seen = torch.arange(cap, device=q.device) <= last[..., None]
    sl.masked_fill_(~seen[None, :, :, None], neg)
    sl = sl.view(kv, b * t * g, cap)
    top = torch.maximum(sp.amax(-1), sl.amax(-1))
    base = torch.where(top == neg, 0.0, top)[..., None]
    sp.sub_(base).exp_()
    sl = sl.sub_(base).exp_()
    total = sp.sum(-1) + sl.sum(-1)
    o = torch.matmul(sp, pv.permute(1, 0, 2)) + torch.matmul(sl.view(kv, b, t * g, cap), lv.permute(2, 0, 1, 3)).view(kv, -1, d)
    o = o / torch.where(total > 0, total, 1.0)[..., None]
    out = o.view(kv, b, t, g, d).permute(1, 2, 0, 3, 4).reshape(b, t, h * d).to(s["q"].dtype)
    lse = (top + total.log()).view(kv, b, t, g).permute(1, 0, 3, 2).reshape(b, h, t)
    return out, lse


def _plain_rules(s):
    """Logits after every rule ``[B, V]`` in 32 bits."""
    case = s["case"]
    b, v = case["batch"], case["vocab"]
    z = s["logits"].float()
    if s["ids"] is not None:
        ids = s["ids"].long()
        place = torch.arange(ids.shape[1], device=z.device)
        live = place < s["hist_len"][:, None]
        output = live & (place >= s["prompt_len"][:, None])
        zeros = torch.zeros(b, v, dtype=torch.int32, device=z.device)
        seen = zeros.scatter_add(1, ids, live.int()) > 0
        count = zeros.scatter_add(1, ids, output.int())
        r = s["repetition"][:, None]
        z = torch.where(seen, torch.where(z > 0, z / r, z * r), z)
        counted = z - s["frequency"][:, None] * count.float() - s["presence"][:, None]
        z = torch.where(count > 0, counted, z)
    if s["bias_ids"] is not None:
        z = z.scatter_add(1, s["bias_ids"].long(), s["bias_values"])
    if s["mask"] is not None:
        bits = (s["mask"][..., None] >> torch.arange(32, device=z.device)) & 1
        z = z.masked_fill(bits.view(b, -1)[:, :v] == 0, float("-inf"))
    return z


def _plain_choose(z):
    value = z.amax(-1)
    index = torch.arange(z.shape[1], device=z.device)
    token = torch.where(z == value[:, None], index, z.shape[1]).amin(-1)
    return torch.where(value == float("-inf"), -1, token), value


def run(state):
    case, op = state["case"], state["case"]["op"]
    if own:
        return _run_own(state, case, op)
    if op in ("rotary", "rotary_cache"):
        return _plain_rotary(state)
    if op == "prefix":
        return _plain_prefix(state)
    z = _plain_rules(state)
    return z.to(state["logits"].dtype) if op == "process" else _plain_choose(z)


# ---------------------------------------------------------------------------------- the framework's operators

def _run_own(s, case, op):
    if op in ("rotary", "rotary_cache"):
        from pdattention_b200.ops.rotary import RotaryTable, rotary, rotary_cache

        table = RotaryTable(s["cos"], s["sin"], interleaved=case["layout"] == "interleaved")
        if op == "rotary_cache":
            q = rotary_cache(s["qkv"], case["heads"], case["kv_heads"], case["dim"], s["positions"], table,
                             s["k_cache"], s["v_cache"], s["slots"])
            return q, s["k_cache"], s["v_cache"]
        out = rotary(s["q"], s["k"], s["positions"], table)
        if not case["grad"]:
            return list(out)
        return [*(t.detach() for t in out), *torch.autograd.grad(out, (s["q"], s["k"]), (s["dq"], s["dk"]))]
    if op == "prefix":
        from pdattention_b200.inference.shared_prefix import shared_prefix_attention

        return shared_prefix_attention(s["q"], s["pk"], s["pv"], s["k"], s["v"], s["lengths"], case["heads"],
                                       case["kv_heads"], case["dim"], prefix_lengths=s["prefix_lengths"], return_lse=True)
    from pdattention_b200.inference.logits import LogitsRules, TokenHistory, choose_tokens, process_logits

    rules = LogitsRules(repetition=s["repetition"], presence=s["presence"], frequency=s["frequency"],
                        bias_ids=s["bias_ids"], bias_values=s["bias_values"], mask=s["mask"])
    history = TokenHistory(s["ids"], s["hist_len"], s["prompt_len"]) if s["ids"] is not None else None
    if op == "process":
        return process_logits(s["logits"], rules, history)
    return choose_tokens(s["logits"], rules, history)


# ---------------------------------------------------------------------------------- the definition in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    with torch.no_grad():
        if op in ("rotary", "rotary_cache"):
            return _exact_rotary(s, case)
        if op == "prefix":
            return _exact_prefix(s, case)
        return _exact_rules(s, case)


def _exact_rotary(s, case):
    n, h, kv, d, rot = (case[k] for k in ("tokens", "heads", "kv_heads", "dim", "rot"))
    pair = torch.arange(rot // 2, device="cuda", dtype=torch.float64)
    freq = torch.exp(-math.log(500000.0) * pair / (rot // 2)) / case["factor"]
    turn = torch.polar(torch.ones_like(freq), s["positions"].double()[:, None] * freq)[:, None]  # e^{i pos f}

    def spin(x, unit):
        x = x.detach().double()
        head, tail = x[..., :rot], x[..., rot:]
        if case["layout"] == "interleaved":
            w = torch.view_as_complex(head.reshape(*head.shape[:-1], rot // 2, 2).contiguous()) * unit
            head = torch.view_as_real(w).flatten(-2)
        else:
            w = torch.complex(head[..., : rot // 2].contiguous(), head[..., rot // 2:].contiguous()) * unit
            head = torch.cat([w.real, w.imag], -1)
        return torch.cat([head, tail], -1)

    if case["op"] == "rotary":
        out = [spin(s["q"], turn), spin(s["k"], turn)]
        return out + [spin(s["dq"], turn.conj()), spin(s["dk"], turn.conj())] if case["grad"] else out
    q, k, v = s["qkv"].view(n, -1, d).split([h, kv, kv], 1)
    kc, vc = s["k_cache"].double(), s["v_cache"].double()
    live = torch.nonzero(s["slots"] >= 0).flatten()
    kc.index_copy_(0, s["slots"][live].long(), spin(k, turn).reshape(n, -1)[live])
    vc.index_copy_(0, s["slots"][live].long(), v.double().reshape(n, -1)[live])
    return spin(q, turn).reshape(n, -1), kc, vc


def _exact_prefix(s, case):
    b, t, h, kv, d, p = (case[k] for k in ("batch", "tokens", "heads", "kv_heads", "dim", "prefix"))
    g, out, lse = h // kv, [], []
    lengths = s["lengths"].tolist()
    shared = s["prefix_lengths"].tolist() if s["prefix_lengths"] is not None else [p] * b
    for row in range(b):
        n, m = lengths[row], shared[row]
        keys = torch.cat([s["pk"][:m], s["k"][row, :n]]).double().view(m + n, kv, d).transpose(0, 1)
        values = torch.cat([s["pv"][:m], s["v"][row, :n]]).double().view(m + n, kv, d).transpose(0, 1)
        q = s["q"][row].double().view(t, kv, g, d)
        hidden = torch.arange(m + n, device="cuda") > m + n - t + torch.arange(t, device="cuda")[:, None]
        for j in range(kv):  # scores of one key/value head at a time: a long suffix's would not all fit in 64 bits
            score = torch.einsum("tgd,nd->tgn", q[:, j], keys[j]) * d ** -0.5
            score.masked_fill_(hidden[:, None], -math.inf)
            total = torch.logsumexp(score, -1)
            weight = torch.exp(score - torch.nan_to_num(total, neginf=0.0)[..., None])
            out.append(torch.einsum("tgn,nd->tgd", weight, values[j]))
            lse.append(total)
    o = torch.stack(out).view(b, kv, t, g, d).transpose(1, 2).reshape(b, t, h * d)
    return o, torch.stack(lse).view(b, kv, t, g).transpose(2, 3).reshape(b, h, t)


def _exact_rules(s, case):
    b, v = case["batch"], case["vocab"]
    rows = []
    for row in range(b):
        z = s["logits"][row].double()
        if s["ids"] is not None:
            ids = s["ids"][row, : int(s["hist_len"][row])].long()
            met = torch.unique(ids)
            z[met] = torch.where(z[met] > 0, z[met] / s["repetition"][row].double(), z[met] * s["repetition"][row].double())
            said, times = torch.unique(ids[int(s["prompt_len"][row]):], return_counts=True)
            z[said] -= s["frequency"][row].double() * times + s["presence"][row].double()
        if s["bias_ids"] is not None:
            z.index_add_(0, s["bias_ids"][row].long(), s["bias_values"][row].double())
        if s["mask"] is not None:
            token = torch.arange(v, device="cuda")
            word = s["mask"][row][token // 32].long()
            z[torch.bitwise_right_shift(word, token % 32) % 2 == 0] = -math.inf
        rows.append(z)
    z = torch.stack(rows)
    return z if case["op"] == "process" else (None, z.max(-1).values)
