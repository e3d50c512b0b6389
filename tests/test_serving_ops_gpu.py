"""Rotary positions, shared-prefix attention and logits rules on the GPU against plain forms in 64 bits.

Tolerances are counted from the roundings: half a step of the output type relative to the value
(``finfo.eps / 2``), half a step of bf16 for each softmax weight (the products take 16-bit weights), and the
fp32 sums (``D * 2^-24`` of the sum of absolute products).
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
NEG = float("-inf")


@pytest.fixture(scope="module", autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.skip("CUDA device required")


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


# ---------------------------------------------------------------------------------- rotary

def rotate64(x, positions, table, inverse=False):
    """``x`` ``[..., H, D]`` in 64 bits, the table's entries as they are."""
    rot, c, s = table.rotary_dim, table.cos.double()[positions][..., None, :], table.sin.double()[positions][..., None, :]
    if inverse:
        s = -s
    x = x.double()
    y = x.clone()
    if table.interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., : rot // 2], x[..., rot // 2: rot]
        y[..., : rot // 2], y[..., rot // 2: rot] = a * c - b * s, b * c + a * s
    return y


def rotary_close(got, want, x, rot):
    # products and sum in fp32 (three roundings of at most |x0| + |x1| <= 2 max), one rounding to the type
    slack = 3 * 2.0 ** -24 * 2 * x.double().abs().amax(-1, keepdim=True)
    assert ((got.double() - want).abs() <= half_step(got.dtype) * want.abs() + slack).all()
    assert torch.equal(got[..., rot:], x[..., rot:])  # what is not rotated passes through


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens,heads,kv,dim,rot", [(1, 1, 1, 64, 64), (5, 3, 1, 64, 32), (37, 8, 2, 128, 128),
                                                      (700, 32, 8, 128, 64), (13, 4, 4, 80, 20), (9, 7, 1, 6, 2),
                                                      (3, 5, 5, 96, 18), (2, 300, 4, 64, 64)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_forward_and_gradient(dtype, tokens, heads, kv, dim, rot, interleaved):
    from pdattention_b200.ops.rotary import rotary, rotary_table

    torch.manual_seed(tokens + rot)
    table = rotary_table(rot, 500, theta=10000.0, interleaved=interleaved, device=DEV)
    q = torch.randn(tokens, heads, dim, device=DEV).to(dtype).requires_grad_()
    k = torch.randn(tokens, kv, dim, device=DEV).to(dtype).requires_grad_()
    pos = torch.randint(0, 500, (tokens,), device=DEV)
    y, z = rotary(q, k, pos, table)
    rotary_close(y, rotate64(q.detach(), pos, table), q.detach(), rot)
    rotary_close(z, rotate64(k.detach(), pos, table), k.detach(), rot)
    dy, dz = torch.randn_like(y), torch.randn_like(z)
    dq, dk = torch.autograd.grad((y, z), (q, k), (dy, dz))
    rotary_close(dq, rotate64(dy, pos, table, inverse=True), dy, rot)
    rotary_close(dk, rotate64(dz, pos, table, inverse=True), dz, rot)


def test_rotary_gradient_against_differences():
    from pdattention_b200.ops.rotary import rotary, rotary_table

    torch.manual_seed(0)
    table = rotary_table(8, 40, theta=100.0, device=DEV)
    q = torch.randn(2, 3, 2, 12, device=DEV, requires_grad=True)
    pos = torch.randint(0, 40, (2, 3), device=DEV, dtype=torch.int32)
    w = torch.randn_like(q)
    loss = lambda x: (rotary(x, None, pos, table)[0].sin() * w).double().sum()  # noqa: E731
    (grad,) = torch.autograd.grad(loss(q), q)
    step, at = 1e-2, [(0, 0, 0, 0), (1, 2, 1, 5), (0, 1, 0, 7), (1, 0, 1, 11)]
    with torch.no_grad():
        for i in at:
            hi, lo = q.clone(), q.clone()
            hi[i] += step
            lo[i] -= step
            # central difference: error step^2 / 6 times the third derivative (|w| times up to 2 sums of
            # products of the rotation, at most 2 |w|_max), and fp32 roundings over 2 step
            slack = step ** 2 / 3 * float(w.abs().max()) + 2.0 ** -20 / step * float(w.abs().max())
            assert abs((loss(hi) - loss(lo)) / (2 * step) - grad[i]) <= slack


def test_rotary_strided_views_broadcast_gradients_and_second_order():
    from pdattention_b200.ops.rotary import rotary, rotary_table

    torch.manual_seed(1)
    table = rotary_table(64, 64, device=DEV)
    qkv = torch.randn(2, 9, 3 * 4 * 64, device=DEV).bfloat16()
    q, k = qkv[..., :256].unflatten(-1, (4, 64)), qkv[..., 256:512].unflatten(-1, (4, 64))
    pos = torch.arange(9, device=DEV).expand(2, 9).contiguous()
    y, z = rotary(q, k, pos, table)
    rotary_close(y, rotate64(q, pos, table), q, 64)
    rotary_close(z, rotate64(k, pos, table), k, 64)
    t = q.transpose(0, 1)  # leading dimensions that do not collapse
    y2, _ = rotary(t, None, pos.t().contiguous(), table)
    assert torch.equal(y2, y.transpose(0, 1))
    shared = torch.randn(1, 9, 4, 64, device=DEV, requires_grad=True)  # one tensor rotated at two offsets
    both, none = rotary(shared.expand(2, 9, 4, 64), None, torch.stack([pos[0], pos[0] + 7]), table)
    assert none is None
    (g,) = torch.autograd.grad(both.sum(), shared)
    ones = torch.ones(1, 9, 4, 64, device=DEV)
    want = sum(rotate64(ones, pos[:1] + d, table, inverse=True) for d in (0, 7))
    assert ((g.double() - want).abs() <= 2.0 ** -22 * 4).all()
    x = torch.randn(3, 2, 64, device=DEV, requires_grad=True)
    p3 = torch.tensor([1, 5, 63], device=DEV)
    y, _ = rotary(x, None, p3, table)
    (g,) = torch.autograd.grad(y.pow(2).sum(), x, create_graph=True)  # |y|^2 = |x|^2: gradient 2 x
    (gg,) = torch.autograd.grad(g.sum(), x)
    assert ((gg - 2).abs() <= 2.0 ** -19).all()


def test_rotary_only_one_gradient_and_bad_positions():
    from pdattention_b200.ops.rotary import rotary, rotary_table

    table = rotary_table(64, 16, device=DEV)
    q = torch.randn(4, 2, 64, device=DEV, requires_grad=True)
    k = torch.randn(4, 1, 64, device=DEV, requires_grad=True)
    pos = torch.tensor([0, 3, 15, 7], device=DEV)
    y, z = rotary(q, k, pos, table)
    (dk,) = torch.autograd.grad(z.sum(), k)
    assert ((dk.double() - rotate64(torch.ones_like(k), pos, table, True)).abs() <= 2.0 ** -21).all()
    wide = torch.cat([q.detach(), q.detach()], -1)  # 64 of 128 rotated
    bad = torch.tensor([0, -1, 16, 7], device=DEV)
    out, _ = rotary(wide, None, bad, table)
    assert out[1:3, :, :64].isnan().all() and torch.equal(out[1:3, :, 64:], wide[1:3, :, 64:])
    rotary_close(out[[0, 3]], rotate64(wide[[0, 3]], bad[[0, 3]], table), wide[[0, 3]], 64)
    e = torch.empty(0, 2, 64, device=DEV)
    assert rotary(e, e[:, :1], torch.empty(0, device=DEV, dtype=torch.long), table)[1].shape == (0, 1, 64)


def test_rotary_backward_in_a_captured_graph():
    """Forward and backward captured, then replayed on other gradients and positions.  (No eager graph of the
    same leaves may be alive then: their accumulation nodes belong to the stream of that graph.)"""
    from pdattention_b200.ops.rotary import rotary, rotary_table

    torch.manual_seed(6)
    table = rotary_table(32, 50, interleaved=True, device=DEV)
    q = torch.randn(11, 3, 64, device=DEV, requires_grad=True)
    k = torch.randn(11, 1, 64, device=DEV, requires_grad=True)
    pos = torch.randint(0, 50, (11,), device=DEV)
    w = torch.randn_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # warm-up on a side stream, as captures want
        torch.autograd.grad((rotary(q, k, pos, table)[0] * w).sum(), q)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, z = rotary(q, k, pos, table)
        dq, dk = torch.autograd.grad((y * w).sum() + z.sum(), (q, k))
    with torch.no_grad():
        w.mul_(2)
        pos.add_(-1).clamp_(min=0)
    graph.replay()
    want = torch.autograd.grad((rotary(q, k, pos, table)[0] * w).sum(), q)[0]
    assert torch.equal(dq, want)
    assert ((dk.double() - rotate64(torch.ones_like(k), pos, table, True)).abs() <= 2.0 ** -21).all()


@pytest.mark.parametrize("tokens,heads,kv,dim,rot,interleaved", [(1, 8, 2, 64, 64, False), (77, 28, 4, 128, 128, False),
                                                                  (300, 12, 12, 64, 32, True), (5, 3, 1, 128, 18, False)])
def test_rotary_cache(tokens, heads, kv, dim, rot, interleaved):
    from pdattention_b200.ops.rotary import rotary_cache, rotary_table

    torch.manual_seed(2)
    table = rotary_table(rot, 300, interleaved=interleaved, device=DEV)
    qkv = torch.randn(tokens, (heads + 2 * kv) * dim + 16, device=DEV).bfloat16()
    rows = tokens + 6
    cache = torch.randn(rows, 2 * kv * dim, device=DEV).bfloat16()
    before = cache.clone()
    slots = torch.randperm(rows, device=DEV)[:tokens].int()
    slots[tokens // 2] = rows if tokens % 2 else -1  # padding, or past the cache: nothing written
    pos = torch.randint(0, 300, (tokens,), device=DEV, dtype=torch.int32)
    q = rotary_cache(qkv, heads, kv, dim, pos, table, cache[:, : kv * dim], cache[:, kv * dim:], slots)
    x = qkv[:, : (heads + 2 * kv) * dim].unflatten(1, (heads + 2 * kv, dim))
    want = rotate64(x[:, : heads + kv], pos.long(), table)
    rotary_close(q.unflatten(1, (heads, dim)), want[:, :heads], x[:, :heads], rot)
    live = ((slots >= 0) & (slots < rows)).nonzero().flatten()
    at = slots[live].long()
    rotary_close(cache[at, : kv * dim].unflatten(1, (kv, dim)), want[live, heads:], x[live, heads: heads + kv], rot)
    assert torch.equal(cache[at, kv * dim:], x[live, heads + kv:].flatten(1))
    other = torch.ones(rows, dtype=torch.bool, device=DEV)
    other[at] = False
    assert torch.equal(cache[other], before[other])


# ---------------------------------------------------------------------------------- shared prefix

def prefix64(q, pk, pv, k, v, lengths, prefix_lengths, heads, kv, dim, scale):
    """Out, lse and, for the tolerances, sum_j p_j |v_j| / sum and the largest sum of absolute products."""
    B, T, _ = q.shape
    g = heads // kv
    out, lse, mass, size = (torch.zeros(*s, dtype=torch.float64, device=DEV) for s in
                            ((B, T, heads, dim), (B, heads, T), (B, T, heads, dim), (B, heads, T)))
    for b in range(B):
        n = min(max(int(lengths[b]), 0), k.shape[1])
        m = pk.shape[0] if prefix_lengths is None else min(max(int(prefix_lengths[b]), 0), pk.shape[0])
        keys = torch.cat([pk[:m], k[b, :n]]).double()[:, : kv * dim].view(m + n, kv, dim).repeat_interleave(g, 1)
        vals = torch.cat([pv[:m], v[b, :n]]).double()[:, : kv * dim].view(m + n, kv, dim).repeat_interleave(g, 1)
        x = q[b].double().view(T, heads, dim)
        s = torch.einsum("thd,nhd->htn", x, keys) * scale
        own = torch.arange(n, device=DEV) <= n - T + torch.arange(T, device=DEV)[:, None]
        seen = torch.cat([torch.ones(T, m, dtype=torch.bool, device=DEV), own], 1)
        s = s.masked_fill(~seen[None], NEG)
        lse[b] = torch.logsumexp(s, -1) if m + n else NEG
        p = torch.exp(s - lse[b].nan_to_num(neginf=0.0)[..., None])
        out[b] = torch.einsum("htn,nhd->thd", p, vals)
        mass[b] = torch.einsum("htn,nhd->thd", p, vals.abs())
        if m + n:
            size[b] = torch.einsum("thd,nhd->htn", x.abs(), keys.abs()).amax(-1) * scale
    return out.flatten(2), lse, mass.flatten(2), size


def prefix_close(got, lse, want, dim):
    out, lse64, mass, size = want
    assert torch.equal(lse == NEG, lse64 == NEG)
    some = lse64 != NEG
    # scores: dim products summed in fp32; exp2 and its argument, the sum of the weights and the logarithm
    slack = dim * 2.0 ** -24 * size + 2.0 ** -20 * (1 + size + lse64.nan_to_num(neginf=0).abs())
    assert ((lse.double() - lse64).abs()[some] <= slack[some]).all()
    # every weight half a step of bf16 and the score's error, the result half a step
    err = (half_step(torch.bfloat16) + 2 * slack.amax()) * mass + half_step(torch.bfloat16) * out.abs() * (1 + 2.0 ** -7)
    assert ((got.double() - out).abs() <= err + 1e-30).all()


CASES = [
    # B, T, P, capacity, H, Hkv, D: decode, drafts, suffixes; one key, one block, ends inside blocks
    (1, 1, 1, 1, 1, 1, 64), (2, 1, 1, 3, 4, 2, 128), (3, 1, 128, 64, 8, 2, 64), (5, 1, 129, 130, 8, 2, 128),
    (9, 1, 1000, 70, 28, 4, 128), (64, 1, 700, 100, 32, 8, 128), (70, 1, 517, 33, 32, 8, 64), (40, 1, 300, 20, 28, 4, 64),
    (7, 5, 333, 90, 12, 12, 64), (4, 3, 260, 17, 32, 4, 128), (2, 70, 400, 150, 8, 2, 128), (3, 129, 77, 200, 4, 4, 64),
    (2, 300, 257, 300, 8, 2, 128), (1, 1, 5000, 10, 32, 8, 128), (1, 513, 900, 600, 4, 1, 64), (2, 40, 130, 64, 64, 2, 64),
    (3, 1, 0, 200, 8, 2, 128), (3, 4, 0, 200, 8, 2, 64), (3, 2, 300, 0, 8, 2, 128), (33, 1, 150, 40, 40, 2, 128),
    (3, 1, 200, 50, 3, 1, 128), (5, 3, 700, 9, 3, 3, 128), (1, 2, 65, 7, 5, 5, 128),  # odd counts of partials
    # more tiles than fit in whole waves of CTAs, or less than one: those behind are split
    (20, 300, 700, 300, 8, 8, 64), (4, 300, 7000, 300, 16, 8, 128), (300, 64, 500, 0, 4, 2, 64),
]


@pytest.mark.parametrize("B,T,P,cap,H,Hkv,D", CASES)
@pytest.mark.parametrize("ragged", [False, True])
def test_shared_prefix_attention(B, T, P, cap, H, Hkv, D, ragged):
    from pdattention_b200.inference.shared_prefix import shared_prefix_attention

    torch.manual_seed(B * 1000 + T + P)
    w = Hkv * D
    q = (1.5 * torch.randn(B, T, H * D, device=DEV)).bfloat16()
    prefix = torch.randn(P, 2 * w, device=DEV).bfloat16()  # keys and values side by side: strided rows
    cache = torch.randn(2, B, cap, w, device=DEV).bfloat16()
    lengths = torch.full((B,), cap, dtype=torch.int32, device=DEV)
    prefix_lengths = None
    if ragged:
        lengths = torch.randint(0, cap + 1, (B,), device=DEV, dtype=torch.int32)
        prefix_lengths = torch.randint(0, P + 1, (B,), device=DEV, dtype=torch.int32)
        if B > 1:
            lengths[0], prefix_lengths[0] = 0, 0  # a row that sees nothing
        # what no query sees may hold anything
        for b in range(B):
            cache[:, b, int(lengths[b]):] = float("nan")
        prefix[int(prefix_lengths.max()):] = float("inf")
    pk, pv = prefix[:, :w], prefix[:, w:]
    out, lse = shared_prefix_attention(q, pk, pv, cache[0], cache[1], lengths, H, Hkv, D,
                                       prefix_lengths=prefix_lengths, return_lse=True)
    want = prefix64(q, pk, pv, cache[0], cache[1], lengths, prefix_lengths, H, Hkv, D, 1 / math.sqrt(D))
    prefix_close(out, lse, want, D)
    from pdattention_b200.ops import _ext
    assert int(_ext.require().attention_status(0)) == 0


@pytest.mark.parametrize("T", [1, 3, 260])
def test_shared_prefix_attention_views_lengths_and_scale(T):
    """Caches inside larger buffers, q inside a fused projection, lengths past the capacity or negative,
    a scale, peaked scores."""
    from pdattention_b200.inference.shared_prefix import shared_prefix_attention

    torch.manual_seed(T)
    B, P, cap, H, Hkv, D = 4, 300, 290, 8, 2, 64
    w = Hkv * D
    fused = torch.randn(B, T, (H + 2 * Hkv) * D, device=DEV).bfloat16()
    q = fused[..., : H * D]
    big = torch.randn(2, B, cap + 14, 2 * w, device=DEV).bfloat16()
    k, v = big[0, :, 9: 9 + cap, w:], big[1, :, 9: 9 + cap, :w]
    pk, pv = torch.randn(2, P, w, device=DEV).bfloat16()
    lengths = torch.tensor([cap + 50, -3, 77, 290], dtype=torch.int32, device=DEV)
    out, lse = shared_prefix_attention(q, pk, pv, k, v, lengths, H, Hkv, D, scale=0.9, return_lse=True)
    prefix_close(out, lse, prefix64(q, pk, pv, k, v, lengths, None, H, Hkv, D, 0.9), D)
    assert torch.equal(shared_prefix_attention(q, pk, pv, k, v, lengths, H, Hkv, D, scale=0.9), out)


@pytest.mark.parametrize("B,T,P,lo,hi,H,Hkv,D", [(78, 1, 2170, 1, 66, 28, 4, 128), (64, 1, 8192, 64, 700, 32, 8, 128),
                                                 (150, 1, 900, 1, 64, 16, 8, 128), (48, 3, 1500, 3, 90, 8, 2, 64),
                                                 (40, 5, 3000, 5, 200, 32, 8, 64), (3, 512, 5000, 512, 600, 32, 8, 128)])
def test_shared_prefix_attention_repeats_exactly(B, T, P, lo, hi, H, Hkv, D):
    """Both parts at once, many short rows to a CTA: every call gives the same bits, and the right ones."""
    from pdattention_b200.inference.shared_prefix import shared_prefix_attention

    torch.manual_seed(P)
    w = Hkv * D
    q = (1.5 * torch.randn(B, T, H * D, device=DEV)).bfloat16()
    pk, pv = torch.randn(2, P, w, device=DEV).bfloat16()
    k, v = torch.randn(2, B, hi + 3, w, device=DEV).bfloat16()
    lengths = torch.tensor([lo + (hi - lo) * i // (B - 1) for i in range(B)], dtype=torch.int32, device=DEV)[torch.randperm(B, device=DEV)]
    run = lambda: shared_prefix_attention(q, pk, pv, k, v, lengths, H, Hkv, D, return_lse=True)  # noqa: E731
    first = run()
    prefix_close(*first, prefix64(q, pk, pv, k, v, lengths, None, H, Hkv, D, 1 / math.sqrt(D)), D)
    again = [run() for _ in range(20)]
    assert all(torch.equal(a, b) for r in again for a, b in zip(r, first))


@pytest.mark.parametrize("B,T,H", [(6, 1, 8), (6, 9, 8), (50, 1, 8), (40, 260, 4)])
def test_shared_prefix_attention_streams_and_graphs(B, T, H):
    from pdattention_b200.inference.shared_prefix import shared_prefix_attention

    torch.manual_seed(5)
    P, cap, Hkv, D = 400, 64, 2, 128
    mk = lambda s: (torch.randn(B, T, H * D, device=DEV).bfloat16(), *torch.randn(2, P, Hkv * D, device=DEV).bfloat16(),  # noqa: E731
                    *torch.randn(2, B, cap, Hkv * D, device=DEV).bfloat16(),
                    torch.randint(1, cap + 1, (B,), device=DEV, dtype=torch.int32))
    one, two = mk(0), mk(1)
    run = lambda a: shared_prefix_attention(*a, H, Hkv, D, return_lse=True)  # noqa: E731
    want = [run(one), run(two)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # two calls at once
        other = [run(two) for _ in range(4)]
    here = [run(one) for _ in range(4)]
    torch.cuda.synchronize()
    for o, h in zip(other, here):
        assert all(torch.equal(x, y) for x, y in zip(o + h, want[1] + want[0]))
    graphs = []
    for a in (one, two):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r = run(a)
        graphs.append((g, r))
    for _ in range(3):
        for g, _ in graphs:
            g.replay()
    torch.cuda.synchronize()
    for (_, r), w in zip(graphs, want):
        assert all(torch.equal(x, y) for x, y in zip(r, w))
    one[5].fill_(3)  # lengths are read when the graph runs
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1][0], run(one)[0]) and not torch.equal(graphs[0][1][0], want[0][0])


# ---------------------------------------------------------------------------------- rules on logits

def rules64(logits, r, history, vocab_start=0):
    """Processed logits in 64 bits, and what their fp32 roundings scale with."""
    z = logits.double().clone()
    size = z.abs().nan_to_num(posinf=0.0)
    B, V = z.shape
    for b in range(B):
        if history is not None:
            n = min(max(int(history.lengths[b]), 0), history.ids.shape[1])
            p = 0 if history.prompt_lengths is None else int(history.prompt_lengths[b])
            ids = history.ids[b, :n].tolist()
            counts = {}
            for i, t in enumerate(ids):
                t -= vocab_start
                if 0 <= t < V:
                    counts[t] = counts.get(t, 0) + (i >= p)
            for t, c in counts.items():
                if r.repetition is not None:
                    f = float(r.repetition[b])
                    z[b, t] = z[b, t] / f if z[b, t] > 0 else z[b, t] * f
                    size[b, t] = torch.maximum(size[b, t], z[b, t].abs().nan_to_num(posinf=0.0))
                if c:
                    cut = (float(r.frequency[b]) * c if r.frequency is not None else 0) + (float(r.presence[b]) if r.presence is not None else 0)
                    z[b, t] -= cut
                    size[b, t] += abs(cut)
        if r.bias_ids is not None:
            for t, x in zip(r.bias_ids[b].tolist(), r.bias_values[b].tolist()):
                if 0 <= t - vocab_start < V:
                    z[b, t - vocab_start] += x
                    size[b, t - vocab_start] += abs(x)
        if r.mask is not None:
            row = b if r.mask_rows is None else int(r.mask_rows[b])
            if row >= r.mask.shape[0]:
                z[b] = NEG
            elif row >= 0:
                t = torch.arange(V, device=DEV) + vocab_start
                bit = (r.mask[row].long()[t // 32] >> (t % 32)) & 1
                z[b] = z[b].masked_fill(bit == 0, NEG)
    return z, size


def make_rules(B, V, hist, biases, mask, seed=0):
    from pdattention_b200.inference.logits import LogitsRules, TokenHistory

    g = torch.Generator(device=DEV).manual_seed(seed)
    rand = lambda *s: torch.rand(*s, generator=g, device=DEV)  # noqa: E731
    r = LogitsRules(repetition=1 + rand(B), presence=rand(B), frequency=rand(B) - 0.3)
    h = None
    if hist:
        ids = (V * rand(B, hist) ** 3).int()
        ids[0, 0] = -1          # ids outside the vocabulary are skipped
        ids[-1, -1] = V + 5
        h = TokenHistory(ids, torch.randint(0, hist + 1, (B,), generator=g, device=DEV).int(),
                         torch.randint(0, hist + 1, (B,), generator=g, device=DEV).int())
        h.lengths[-1] = hist + 9  # clamped to the capacity
    if biases:
        r.bias_ids = (V * rand(B, biases)).int()
        r.bias_ids[:, -1] = r.bias_ids[:, 0]  # a token listed twice gets the sum
        r.bias_ids[0, biases // 2] = -1
        r.bias_values = 4 * rand(B, biases) - 2
    if mask:
        words = (V + 31) // 32
        r.mask = torch.randint(-2 ** 31, 2 ** 31, (3, words), generator=g, device=DEV).int()
        r.mask[1] = 0  # allows nothing
        r.mask_rows = (torch.arange(B, device=DEV) % 5 - 1).int()  # -1: none, 0 .. 2, 3: past the masks
    return r, h


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,V,hist,biases,mask", [(1, 1, 3, 0, False), (2, 31, 5, 3, True), (6, 1000, 0, 0, True),
                                                  (5, 4099, 64, 300, True), (3, 32768, 2000, 0, False),
                                                  (4, 50257, 100, 17, True), (7, 128256, 700, 40, True),
                                                  (2, 5000, 30001, 2047, True), (1, 393216, 60000, 2047, False),
                                                  (150, 2000, 1500, 2, True), (150, 2500, 30, 0, False)])
def test_process_and_choose(dtype, B, V, hist, biases, mask):
    from pdattention_b200.inference.logits import choose_tokens, process_logits

    torch.manual_seed(V)
    logits = (2.5 * torch.randn(B, V, device=DEV)).to(dtype)
    logits[0, 0] = float("inf")
    logits[-1, V // 2] = NEG
    r, h = make_rules(B, V, hist, biases, mask)
    before = logits.clone()
    got = process_logits(logits, r, h)
    want, size = rules64(logits, r, h)
    assert torch.equal(logits, before) and got.dtype == dtype
    finite = want.isfinite()
    assert torch.equal(got.double()[~finite], want[~finite])
    slack = 6 * 2.0 ** -24 * size + half_step(dtype) * want.abs() * (1 + 2.0 ** -7)
    assert ((got.double() - want).abs()[finite] <= slack[finite]).all()
    # the choice is the lowest id of the largest processed logit, in 32 bits
    wide = process_logits(logits.float(), r, h)
    if dtype == torch.float32:
        assert torch.equal(wide, got)
    token, value = choose_tokens(logits, r, h)
    best = wide.max(1).values
    first = torch.where(wide == best[:, None], torch.arange(V, device=DEV), V).min(1).values
    assert torch.equal(value, best)
    assert torch.equal(token, torch.where(best == NEG, -1, first))
    inplace = process_logits(logits, r, h, out=logits)
    assert inplace is logits or inplace.data_ptr() == logits.data_ptr()
    assert torch.equal(logits, got)


def test_logits_views_slices_and_special_values():
    from pdattention_b200.inference.logits import LogitsRules, choose_tokens, process_logits

    torch.manual_seed(3)
    B, V = 4, 1003
    big = torch.randn(B, V + 30, device=DEV).bfloat16()
    r, h = make_rules(B, V, 50, 9, True)
    whole = process_logits(big[:, :V].contiguous(), r, h)
    for start in (0, 8, 16):  # unaligned rows, odd strides, slices of the vocabulary
        part = big[:, start: start + 501]
        got = process_logits(part, r, h, vocab_start=start)
        assert torch.equal(got, whole[:, start: start + 501])
        token, value = choose_tokens(part, r, h, vocab_start=start)
        want = process_logits(part.float(), r, h, vocab_start=start)
        best = want.max(1).values
        first = torch.where(want == best[:, None], torch.arange(501, device=DEV) + start, V).min(1).values
        assert torch.equal(value, best) and torch.equal(token, torch.where(best == NEG, -1, first))
    plain = LogitsRules()
    x = torch.zeros(5, 40, device=DEV)
    x[0, 7] = -0.0                    # equal to the zeros before it
    x[1, 3] = x[1, 30] = 1.0          # a tie
    x[2, 9] = float("nan")
    x[3] = NEG
    x[4, 39] = float("inf")
    token, value = choose_tokens(x, plain)
    assert token.tolist() == [0, 3, 9, -1, 39]
    assert value.tolist()[:2] == [0.0, 1.0] and value[2].isnan() and value[3] == NEG
    masked = LogitsRules(mask=torch.full((5, 2), -1, device=DEV, dtype=torch.int32))
    masked.mask[2, 0] = ~(1 << 9)     # NaN in a masked place
    assert choose_tokens(x, masked)[0][2] == 0
    assert process_logits(x, masked)[2, 9] == NEG
    assert process_logits(torch.empty(0, 40, device=DEV), plain).shape == (0, 40)


def test_logits_repeats_exactly_and_appends_in_a_graph():
    from pdattention_b200.inference.logits import LogitsRules, TokenHistory, choose_tokens

    torch.manual_seed(4)
    B, V = 3, 5000
    logits = torch.randn(B, V, device=DEV)
    prompts = torch.randint(0, V, (B, 6), device=DEV)
    history = TokenHistory.start(prompts, torch.tensor([6, 2, 4]), 4)
    rules = LogitsRules(presence=torch.full((B,), 100.0, device=DEV))
    static = logits.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        token, _ = choose_tokens(static, rules, history, append=True)
    seen = []
    for _ in range(3):  # every replay sees the tokens of the ones before: no token twice
        graph.replay()
        seen.append(token.clone())
    assert history.lengths.tolist() == [9, 5, 7]
    order = logits.argsort(1, descending=True)
    assert torch.equal(torch.stack(seen, 1), order[:, :3])
    for b, n in enumerate([6, 2, 4]):
        assert history.ids[b, n: n + 3].tolist() == order[b, :3].tolist()
    history.append(torch.tensor([1, -1, 2], device=DEV))
    assert history.lengths.tolist() == [10, 5, 8]
    history.append(torch.tensor([3, 3, 3], device=DEV))  # row 0 is full: it keeps what it has
    assert history.lengths.tolist() == [10, 6, 9] and history.ids[0, 9] == 1
    choose_tokens(logits, rules, history, append=True)
    assert history.lengths.tolist() == [10, 7, 10]
    i32 = lambda *s: torch.zeros(*s, device=DEV, dtype=torch.int32)  # noqa: E731
    for rows, capacity in ((0, 4), (2, 0)):  # no rows; no room
        h = TokenHistory(i32(rows, capacity), i32(rows))
        token, _ = choose_tokens(logits[:rows], LogitsRules(), h, append=True)
        assert token.tolist() == logits[:rows].argmax(1).tolist() and h.lengths.tolist() == [0] * rows


# ---------------------------------------------------------------------------------- refusals

def refused(fn, *words):
    with pytest.raises((RuntimeError, ValueError)) as e:
        fn()
    assert any(w in str(e.value) for w in words), str(e.value)


def test_refusals_of_rotary():
    from pdattention_b200.ops.rotary import RotaryTable, rotary, rotary_cache, rotary_table

    t = rotary_table(64, 8, device=DEV)
    q = torch.zeros(3, 2, 64, device=DEV).bfloat16()
    pos = torch.zeros(3, device=DEV, dtype=torch.long)
    refused(lambda: rotary(q.double(), None, pos, t), "dtype")
    refused(lambda: rotary(q, None, pos[:2], t), "leading dimensions")
    refused(lambda: rotary(q, q.float(), pos, t), "dtype")
    refused(lambda: rotary(q[..., :32].contiguous(), None, pos, t), "rotates")
    refused(lambda: rotary(q, None, pos.float(), t), "int32 or int64")
    refused(lambda: rotary(q, None, pos.cpu(), t), "must be on")
    refused(lambda: rotary(q, None, pos, RotaryTable(t.cos.double(), t.sin)), "dtype")
    refused(lambda: rotary(q, None, pos, RotaryTable(t.cos[:0], t.sin[:0])), "no positions")
    qkv, cache = torch.zeros(3, 4 * 64, device=DEV).bfloat16(), torch.zeros(8, 64, device=DEV).bfloat16()
    slots = torch.arange(3, device=DEV, dtype=torch.int32)
    ok = lambda **kw: rotary_cache(**{**dict(qkv=qkv, heads=2, kv_heads=1, head_dim=64, positions=pos, table=t,  # noqa: E731
                                             k_cache=cache, v_cache=cache.clone(), slots=slots), **kw})
    ok()
    refused(lambda: ok(heads=3), "qkv")
    refused(lambda: ok(slots=slots.long()), "dtype")
    refused(lambda: ok(slots=slots[:2]), "entries")
    refused(lambda: ok(k_cache=cache[:, :32]), "caches")
    refused(lambda: ok(v_cache=cache[:4]), "caches")
    refused(lambda: ok(v_cache=cache.float()), "dtype")


def test_partials_join_to_the_same_attention():
    from pdattention_b200.inference.shared_prefix import (merge_attention_partials, shared_prefix_attention,
                                                          shared_prefix_partials)

    torch.manual_seed(9)
    for B, T, P, cap, H, Hkv, D in [(5, 1, 300, 40, 8, 2, 128), (2, 300, 200, 300, 4, 2, 64), (3, 20, 130, 30, 8, 2, 64), (2, 1, 0, 0, 4, 4, 64)]:
        w = Hkv * D
        q = torch.randn(B, T, H * D, device=DEV).bfloat16()
        pk, pv = torch.randn(2, P, w, device=DEV).bfloat16()
        k, v = torch.randn(2, B, cap, w, device=DEV).bfloat16()
        ln = torch.full((B,), cap, dtype=torch.int32, device=DEV)
        args = (q, pk, pv, k, v, ln, H, Hkv, D)
        want = shared_prefix_attention(*args, return_lse=True)
        parts = shared_prefix_partials(*args)
        assert parts[0].shape == (B * T, H, 1, D) and parts[1].shape == (B * T, H, 1, 2)
        out, lse = merge_attention_partials(parts, batch=B, return_lse=True)
        # the same sums, divided by 1 / l in one place or the other: a last place of fp32 before the rounding
        assert ((out.double() - want[0].double()).abs() <= half_step(torch.bfloat16) * 2 * want[0].double().abs() + 1e-30).all()
        assert ((lse - want[1]).nan_to_num().abs() <= 2.0 ** -20 * (1 + want[1].nan_to_num(neginf=0).abs())).all()
        # keys seen twice weigh twice: the same output, log 2 more
        twice, lse2 = merge_attention_partials(parts, parts, batch=B, return_lse=True)
        assert torch.equal(twice, out) and ((lse2 - lse - math.log(2)).nan_to_num().abs() <= 2.0 ** -19 * (1 + lse.nan_to_num(neginf=0).abs())).all()
    refused(lambda: merge_attention_partials((parts[0], parts[1].double()), batch=2), "dtype")
    refused(lambda: merge_attention_partials(parts, batch=3), "whole batch rows")
    refused(lambda: merge_attention_partials((parts[0][..., :32].contiguous(), parts[1]), batch=2), "head_dim")


@pytest.mark.parametrize("B,T,P,cap,bad", [(4, 1, 300, 0, "prefix"), (4, 1, 300, 20, "prefix"), (4, 1, 300, 20, "own"),
                                           (1, 1, 5000, 20, "prefix"), (2, 40, 700, 50, "prefix")])
def test_a_visible_nan_reaches_its_rows(B, T, P, cap, bad):
    """A NaN key that a row sees makes that row NaN, its log sum too, and no other row."""
    from pdattention_b200.inference.shared_prefix import (merge_attention_partials, shared_prefix_attention,
                                                          shared_prefix_partials)

    torch.manual_seed(5)
    H, Hkv, D = 4, 2, 64
    q = torch.randn(B, T, H * D, device=DEV).bfloat16()
    pk, pv = torch.randn(2, P, Hkv * D, device=DEV).bfloat16()
    k, v = torch.randn(2, B, cap, Hkv * D, device=DEV).bfloat16()
    ln = torch.full((B,), cap, dtype=torch.int32, device=DEV)
    see = torch.full((B,), P, dtype=torch.int32, device=DEV)
    if bad == "prefix":
        pk[150:] = float("nan")  # some parts hold nothing but NaN
        see[1:] = 150
        if cap:
            ln[0] = T - 1 if T > 1 else 0
        hit = torch.arange(B, device=DEV) == 0
    else:
        k[-1] = float("nan")
        hit = torch.arange(B, device=DEV) == B - 1
    args = (q, pk, pv, k, v, ln, H, Hkv, D)
    out, lse = shared_prefix_attention(*args, prefix_lengths=see, return_lse=True)
    assert torch.equal(out.isnan().any(-1).all(-1), hit) and torch.equal(out.isnan().all(-1).any(-1), hit)
    assert torch.equal(lse.isnan().flatten(1).all(1), hit) and torch.equal(lse.isnan().flatten(1).any(1), hit)
    o, ml = shared_prefix_partials(*args, prefix_lengths=see)
    out, lse = merge_attention_partials((o, ml), (torch.zeros_like(o), torch.full_like(ml, NEG)), batch=B, return_lse=True)
    assert torch.equal(out.isnan().flatten(1).all(1), hit) and torch.equal(lse.isnan().flatten(1).any(1), hit)


def test_a_part_of_nan_is_no_empty_part():
    from pdattention_b200.inference.shared_prefix import merge_attention_partials

    o = torch.zeros(2, 1, 40, 64, device=DEV)
    ml = torch.full((2, 1, 40, 2), NEG, device=DEV)
    ml[0, 0, 37] = float("nan")
    out, lse = merge_attention_partials((o, ml), batch=2, return_lse=True)
    assert out[0].isnan().all() and lse[0].isnan().all() and (out[1] == 0).all() and (lse[1] == NEG).all()


def test_refusals_of_shared_prefix_attention():
    from pdattention_b200.inference.shared_prefix import shared_prefix_attention

    B, T, P, cap, H, Hkv, D = 2, 1, 10, 12, 4, 2, 64
    z = lambda *s: torch.zeros(*s, device=DEV).bfloat16()  # noqa: E731
    base = dict(q=z(B, T, H * D), prefix_k=z(P, Hkv * D), prefix_v=z(P, Hkv * D), k=z(B, cap, Hkv * D),
                v=z(B, cap, Hkv * D), lengths=torch.ones(B, device=DEV, dtype=torch.int32), heads=H, kv_heads=Hkv,
                head_dim=D)
    ok = lambda **kw: shared_prefix_attention(**{**base, **kw})  # noqa: E731
    ok()
    refused(lambda: ok(q=base["q"].float()), "dtype")
    refused(lambda: ok(k=base["k"].half()), "dtype")
    refused(lambda: ok(head_dim=32, heads=8), "head_dim")
    refused(lambda: ok(heads=3), "multiple")
    refused(lambda: ok(q=z(B, T, H * D - 8)), "q must be")
    refused(lambda: ok(prefix_v=z(P + 1, Hkv * D)), "prefix keys and values")
    refused(lambda: ok(prefix_k=z(P, D), prefix_v=z(P, D)), "at least")
    refused(lambda: ok(k=z(B + 1, cap, Hkv * D)), "own keys and values")
    refused(lambda: ok(lengths=base["lengths"].long()), "dtype")
    refused(lambda: ok(lengths=base["lengths"][:1]), "entries")
    refused(lambda: ok(lengths=base["lengths"].cpu()), "must be on")
    refused(lambda: ok(scale=0.0), "scale")
    refused(lambda: ok(scale=1e-50), "scale")
    refused(lambda: ok(scale=1e50), "scale")
    refused(lambda: ok(prefix_lengths=torch.ones(B, device=DEV)), "dtype")
    refused(lambda: ok(prefix_k=z(P, Hkv * D + 4)[:, : Hkv * D]), "multiples of 16 bytes")
    refused(lambda: ok(prefix_k=z(P * Hkv * D + 1)[1:].view(P, Hkv * D)), "16-byte boundary")
    refused(lambda: ok(k=z(Hkv * D, B, cap).permute(1, 2, 0)), "contiguous rows")
    refused(lambda: ok(k=z(1, cap, Hkv * D).expand(B, -1, -1)), "strides")


def test_refusals_of_logits_rules():
    from pdattention_b200.inference.logits import LogitsRules, TokenHistory, choose_tokens, process_logits

    B, V = 2, 100
    x = torch.zeros(B, V, device=DEV)
    i32 = lambda *s: torch.zeros(*s, device=DEV, dtype=torch.int32)  # noqa: E731
    h = TokenHistory(i32(B, 5), i32(B), i32(B))
    process_logits(x, LogitsRules(), h)
    refused(lambda: process_logits(x.double(), LogitsRules()), "dtype")
    refused(lambda: process_logits(x.t(), LogitsRules()), "contiguous rows")
    refused(lambda: process_logits(x, LogitsRules(), vocab_start=4), "multiple of 8")
    refused(lambda: process_logits(x, LogitsRules(repetition=torch.ones(B, device=DEV).double()), h), "dtype")
    refused(lambda: process_logits(x, LogitsRules(presence=torch.ones(3, device=DEV)), h), "entries")
    refused(lambda: process_logits(x, LogitsRules(), TokenHistory(i32(B, 5).long(), i32(B))), "dtype")
    refused(lambda: process_logits(x, LogitsRules(), TokenHistory(i32(B, 1 << 20), i32(B))), "fewer than")
    refused(lambda: process_logits(x, LogitsRules(bias_ids=i32(B, 3))), "ids and values")
    refused(lambda: process_logits(x, LogitsRules(bias_ids=i32(B, 2048), bias_values=torch.zeros(B, 2048, device=DEV))), "at most")
    refused(lambda: process_logits(x, LogitsRules(mask=i32(B, 3))), "mask must")
    refused(lambda: process_logits(x, LogitsRules(mask=i32(3, 4))), "one mask per row")
    refused(lambda: process_logits(x, LogitsRules(mask_rows=i32(B))), "without a mask")
    refused(lambda: process_logits(x, LogitsRules(), out=x[:, :50]), "shaped as")
    refused(lambda: process_logits(x.view(-1)[:100].view(1, 100), LogitsRules(), out=x.view(-1)[10:110].view(1, 100)), "overlap")
    refused(lambda: process_logits(torch.zeros(1, 384 * 1024 + 8, device=DEV), LogitsRules(), TokenHistory(i32(1, 2), i32(1))), "columns")
    refused(lambda: choose_tokens(x, LogitsRules(), append=True), "append")
    refused(lambda: choose_tokens(x, LogitsRules(), TokenHistory(i32(1, 5).expand(B, -1), i32(B)), append=True), "overlap")
