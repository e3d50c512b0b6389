"""Corner calls of the serving operators on the GPU: waits that ran out, unusual views, empty tables, lifetimes."""

import math

import pytest
import torch

from test_serving_ops_gpu import half_step, prefix64, prefix_close, rotary_close, rotate64

pytestmark = pytest.mark.gpu
DEV = "cuda"
NEG_INF = float("-inf")


@pytest.fixture(scope="module", autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.skip("CUDA device required")


@pytest.mark.parametrize("B,T,P,cap,H,Hkv,D", [(5, 1, 0, 200, 8, 2, 128), (9, 2, 300, 130, 8, 2, 64), (64, 1, 700, 100, 32, 8, 128),
                                               (3, 40, 300, 90, 8, 2, 128), (1, 300, 500, 300, 8, 2, 64)])
def test_waits_that_ran_out_end_in_the_status_word(B, T, P, cap, H, Hkv, D):
    """Every CTA takes the way of one that gave up: the call ends, the status word says so, and the next
    call is right again.  The workspace holds large integers beforehand."""
    from pdattention_b200.inference.shared_prefix import shared_prefix_attention
    from pdattention_b200.ops import _ext

    torch.manual_seed(B)
    ext, w = _ext.require(), Hkv * D
    q = torch.randn(B, T, H * D, device=DEV).bfloat16()
    pk, pv = torch.randn(2, P, w, device=DEV).bfloat16()
    k, v = torch.randn(2, B, cap, w, device=DEV).bfloat16()
    lengths = torch.randint(T, cap + 1, (B,), device=DEV, dtype=torch.int32)
    run = lambda: shared_prefix_attention(q, pk, pv, k, v, lengths, H, Hkv, D, return_lse=True)  # noqa: E731
    status = ext.attention_status(0)
    junk = [torch.full((1 << n,), 0x7F7F7F7F, dtype=torch.int32, device=DEV) for n in range(8, 24)]
    del junk
    ext.prefix_attention_give_up(True)
    try:
        run()
    finally:
        ext.prefix_attention_give_up(False)
    torch.cuda.synchronize()
    assert int(status) == 1
    status.zero_()
    prefix_close(*run(), prefix64(q, pk, pv, k, v, lengths, None, H, Hkv, D, 1 / math.sqrt(D)), D)
    assert int(status) == 0


@pytest.mark.parametrize("copy", [2, 3, 4, 5, 8])
@pytest.mark.parametrize("B,T,P,cap,H,Hkv,D", [(64, 1, 4000, 700, 32, 8, 128), (64, 8, 4000, 700, 8, 2, 64), (5, 300, 3000, 300, 8, 2, 128),
                                               (200, 300, 700, 300, 2, 1, 64)])
def test_giving_up_with_copies_and_products_in_flight(copy, B, T, P, cap, H, Hkv, D):
    """The wait that runs out is the producer's, behind some copies: the other roles still work on what came.
    The CTAs end with nothing in flight, so the next call, on the same SMs, is right."""
    from pdattention_b200.inference.shared_prefix import shared_prefix_attention
    from pdattention_b200.ops import _ext

    torch.manual_seed(copy)
    ext, w = _ext.require(), Hkv * D
    q = torch.randn(B, T, H * D, device=DEV).bfloat16()
    pk, pv = torch.randn(2, P, w, device=DEV).bfloat16()
    k, v = torch.randn(2, B, cap, w, device=DEV).bfloat16()
    lengths = torch.full((B,), cap, device=DEV, dtype=torch.int32)
    run = lambda: shared_prefix_attention(q, pk, pv, k, v, lengths, H, Hkv, D, return_lse=True)  # noqa: E731
    first = run()
    status = ext.attention_status(0)
    assert int(status) == 0
    ext.prefix_attention_give_up(copy)
    try:
        run()
    finally:
        ext.prefix_attention_give_up(0)
    again = run()  # right behind it
    torch.cuda.synchronize()
    assert int(status) == 1
    status.zero_()
    assert all(torch.equal(a, b) for a, b in zip(again, first))


def test_rotary_of_views_with_dimensions_of_one():
    """Sizes of 1 among the leading dimensions, their strides those of a slice or of a permuted tensor."""
    from pdattention_b200.ops.rotary import rotary, rotary_table

    torch.manual_seed(0)
    base = torch.randn(3, 2, 3, 4, 64, device=DEV).bfloat16()
    table = rotary_table(64, 50)
    for x in (base[:, ::2], base[:1].permute(1, 2, 0, 3, 4), base[:, :, ::3], base[:, :1, :1].transpose(0, 2), base.transpose(0, 2)):
        pos = torch.randint(0, 50, x.shape[:-2], device=DEV)
        rotary_close(rotary(x, None, pos, table)[0], rotate64(x, pos, table), x, 64)
        leaf = torch.randn(x.shape, device=DEV).bfloat16().requires_grad_()
        (grad,) = torch.autograd.grad(rotary(leaf, None, pos, table)[0], leaf, x)  # the incoming gradient is such a view
        rotary_close(grad, rotate64(x, pos, table, inverse=True), x, 64)


def test_a_captured_step_keeps_its_rules_and_history():
    """The caller's objects may go, or get other tensors: the graph's are alive until it is released."""
    import weakref

    from test_serving_engine_gpu import setup

    from pdattention_b200.inference.logits import LogitsRules, TokenHistory

    cfg, model, engine = setup(6)
    ids, n = torch.randint(0, cfg.vocab_size, (2, 6)), torch.tensor([6, 3])
    rules = LogitsRules(repetition=torch.full((2,), 1.5, device=DEV), bias_ids=torch.tensor([[3], [5]], device=DEV).int(),
                        bias_values=torch.ones(2, 1, device=DEV))
    history = TokenHistory.start(ids.to(DEV), n, 6)
    tok = engine.prefill(ids, n, 6).float().argmax(-1)
    engine.decode_step(tok, sample=True, rules=rules, history=history)
    engine.capture_decode(sample=True, rules=rules, history=history)
    held = [weakref.ref(t) for t in (rules.repetition, rules.bias_ids, rules.bias_values, history.ids, history.lengths,
                                     history.prompt_lengths)]
    rules.repetition = torch.full((2,), 9.0, device=DEV)
    del rules, history
    assert all(r() is not None for r in held)
    engine.release_graph()
    assert all(r() is None for r in held)


def test_a_capture_before_the_first_routed_step_leaves_eager_steps_right():
    """Memory that comes after the first step, a capture, then an eager step: the same logits as without the capture."""
    from test_serving_engine_gpu import setup

    outs = []
    for capture in (False, True):
        cfg, model, engine = setup(7)
        gen = torch.Generator().manual_seed(7)
        draw = lambda *s: torch.randint(0, cfg.vocab_size, s, generator=gen)  # noqa: E731
        engine.set_shared_prefix(draw(70))
        engine.prefill(draw(2, 9), torch.tensor([9, 4]), 6)
        engine.decode_step(draw(2))
        engine.build_memory(draw(12, 16), torch.full((12,), 16, dtype=torch.int32))
        engine.set_namespace(torch.zeros(2, dtype=torch.int32), torch.full((2,), 12, dtype=torch.int32))
        if capture:
            engine.capture_decode()
            assert engine._no_len.tolist() == [0, 0]
            kept = engine._no_len
        outs.append(engine.decode_step(draw(2)))
        if capture:
            assert engine._no_len is kept  # made with the cache, not while the step was captured
            engine.prefill(draw(2, 9), torch.tensor([9, 4]), 6)
            assert engine._no_len is not kept
    assert torch.equal(*outs)


@pytest.mark.parametrize("biases", [False, True])
def test_an_empty_set_of_masks_allows_nothing(biases):
    """mask [0, words] with mask_rows: every row that names a mask names one that is not there."""
    from pdattention_b200.inference.logits import LogitsRules, choose_tokens, process_logits

    x = torch.randn(3, 100, device=DEV)
    more = dict(bias_ids=torch.tensor([[4]] * 3, device=DEV).int(), bias_values=torch.full((3, 1), 50.0, device=DEV)) if biases else {}
    rules = LogitsRules(mask=torch.empty(0, 4, dtype=torch.int32, device=DEV),
                        mask_rows=torch.tensor([0, -1, 7], dtype=torch.int32, device=DEV), **more)
    want = x.clone()
    if biases:
        want[:, 4] += 50.0
    want[0::2] = float("-inf")
    assert torch.equal(process_logits(x, rules), want)
    token, value = choose_tokens(x, rules)
    assert token.tolist() == [-1, int(want[1].argmax()), -1] and torch.equal(value, want.amax(1))


@pytest.mark.parametrize("P,cap,n", [(0, 0, 0), (0, 5, 0), (3, 0, 0), (300, 40, 0)])
def test_partials_of_queries_that_see_nothing(P, cap, n):
    """Sums 0, maximum -inf, sum of the weights 0, whether keys are there or not."""
    from pdattention_b200.inference.shared_prefix import merge_attention_partials, shared_prefix_partials

    B, T, H, Hkv, D = 2, 3, 4, 2, 64
    junk = torch.full((1 << 16,), float("nan"), device=DEV)
    del junk
    q = torch.randn(B, T, H * D, device=DEV).bfloat16()
    pk, pv = torch.randn(2, P, Hkv * D, device=DEV).bfloat16()
    k, v = torch.randn(2, B, cap, Hkv * D, device=DEV).bfloat16()
    none = torch.full((B,), n, dtype=torch.int32, device=DEV)
    o, ml = shared_prefix_partials(q, pk, pv, k, v, none, H, Hkv, D, prefix_lengths=none)
    assert o.shape == (B * T, H, 1, D) and (o == 0).all()
    assert (ml[..., 0] == float("-inf")).all() and (ml[..., 1] == 0).all()
    out, lse = merge_attention_partials((o, ml), batch=B, return_lse=True)
    assert (out == 0).all() and (lse == float("-inf")).all()


@pytest.mark.parametrize("T", [1, 20])
@pytest.mark.parametrize("P", [0, 90])
def test_one_own_key_at_any_batch_stride(T, P):
    """A capacity of one row: the batch stride is no multiple of the row's width."""
    from pdattention_b200.inference.shared_prefix import shared_prefix_attention

    torch.manual_seed(T)
    B, H, Hkv, D = 5, 8, 2, 64
    w = Hkv * D
    q = torch.randn(B, T, H * D, device=DEV).bfloat16()
    pk, pv = torch.randn(2, P, w, device=DEV).bfloat16()
    k = torch.randn(B, w + 40, device=DEV).bfloat16()[:, None, 8: 8 + w]
    v = torch.randn(B, 2 * w + 8, device=DEV).bfloat16()[:, None, 16: 16 + w]
    lengths = torch.tensor([1, 0, 1, 1, 1], dtype=torch.int32, device=DEV)
    out, lse = shared_prefix_attention(q, pk, pv, k, v, lengths, H, Hkv, D, return_lse=True)
    prefix_close(out, lse, prefix64(q, pk, pv, k, v, lengths, None, H, Hkv, D, 1 / math.sqrt(D)), D)


def test_batch_strides_that_no_tensor_map_takes_are_refused():
    from pdattention_b200.inference.shared_prefix import shared_prefix_attention

    w = 64
    k = torch.zeros(2 * (3 * w + 8), device=DEV).bfloat16().as_strided((2, 3, w), (3 * w + 8, w, 1))
    with pytest.raises(RuntimeError, match="batch stride"):
        shared_prefix_attention(torch.zeros(2, 1, w, device=DEV).bfloat16(), k[0], k[0], k, k,
                                torch.ones(2, dtype=torch.int32, device=DEV), 1, 1, 64)


class Routing:
    """The oracle takes the chunks that the engine took, so that a tie decided by bf16 activations changes no
    logits; each of them must be one of the oracle's best, up to the bound of the engine's tests (a cosine of
    0.995 to the fp32 activations: a query and a gist turned by at most sqrt(2 * 0.005) each)."""

    def __init__(self, engine, monkeypatch):
        from pdattention_b200.models import llama

        self.engine, self.taken, self.row, self.layer = engine, {}, 0, 0
        route, F = engine._route, torch.nn.functional

        def recording(layer, *args, **kw):
            out = route(layer, *args, **kw)
            self.taken.setdefault(layer, []).append(engine.last_selection[layer])
            return out

        def select(cfg, query, gist, namespace):
            taken = [c for c in torch.cat(self.taken[self.layer])[self.row].tolist() if c >= 0]
            score = F.normalize(gist.float(), dim=-1) @ F.normalize(query[0].float(), dim=-1)
            best = score[namespace[0]].topk(cfg.top_k_chunks).values
            assert sorted(set(taken)) == taken and len(taken) == cfg.top_k_chunks
            assert (score[taken] >= best[-1] - 2 * 2 * math.sqrt(2 * 0.005)).all()
            self.layer += 1
            return [taken]

        engine._route = recording
        monkeypatch.setattr(llama, "select_chunks", select)

    def step(self, row):
        self.row, self.layer = row, 0


@pytest.mark.parametrize("prefix,memory,row_batch", [(0, False, None), (0, True, 1), (20, False, None), (60, True, None)])
def test_dynamic_scaling_past_the_window(prefix, memory, row_batch, monkeypatch):
    """Rows of several lengths, each scaled by its own; prefill, eager and replayed steps, against the fp32 oracle."""
    from test_serving_engine_gpu import close, setup

    from pdattention_b200.models.llama import reference_step

    cfg, model, engine = setup(8, chunk_tokens=48,
                               rope_scaling={"rope_type": "dynamic", "factor": 4.0, "original_max_position_embeddings": 32})
    L, B = cfg.num_hidden_layers, 3
    ids, n = torch.randint(0, cfg.vocab_size, (B, 90)), torch.tensor([90, 41, 7])
    ref_mem = ns = None
    if memory:
        chunks, lengths = torch.randint(0, cfg.vocab_size, (12, 48)), torch.randint(20, 49, (12,))
        engine.build_memory(chunks, lengths)  # chunks on both sides of the window
        engine.set_namespace(torch.zeros(B), torch.full((B,), 12))
        ref_mem, ns = model.encode_chunks(chunks, lengths), list(range(12))
    routing = Routing(engine, monkeypatch)
    caches = [[[None, None] for _ in range(L)] for _ in range(B)]
    if prefix:
        head = torch.randint(0, cfg.vocab_size, (prefix,))
        engine.set_shared_prefix(head, chunk_tokens=25)
        for b in range(B):
            reference_step(model, head, caches[b], None, None)
    logits = engine.prefill(ids, n, 8, row_batch=row_batch)
    for b in range(B):
        routing.step(b)
        close(logits[b], reference_step(model, ids[b, : n[b]], caches[b], ref_mem, ns)[0][-1], 0.995)
    for step in range(4):
        routing.taken.clear()
        if step == 2:
            engine.capture_decode()
        tok = torch.randint(0, cfg.vocab_size, (B,))
        got = engine.decode_step(tok) if step < 2 else engine.decode_step_graphed(tok)
        if step == 3:  # nothing is recorded at a replay: the graph's own outputs
            routing.taken.update({layer: [sel] for layer, sel in engine.last_selection.items()})
        for b in range(B):
            routing.step(b)
            close(got[b], reference_step(model, tok[b: b + 1], caches[b], ref_mem, ns)[0][-1], 0.99)
    engine.release_graph()


def test_penalties_see_the_shared_prefix():
    """Repetition that rules a token out for good: what the prefix says is not said again.  Every token is the best
    of the engine's own logits after the penalties of prefix, prompt and output."""
    from test_serving_engine_gpu import setup

    from pdattention_b200.inference.logits import LogitsRules

    cfg, model, engine = setup(9)
    B, new, V = 2, 10, cfg.vocab_size
    ids, n = torch.randint(0, V, (B, 7)), torch.tensor([7, 3])
    engine.set_shared_prefix(torch.arange(0, 40))
    logits = engine.prefill(ids, n, new)
    prefix = torch.cat([torch.arange(0, 40), logits.float().topk(20, dim=-1).indices.flatten().cpu()])  # and the likeliest
    engine.set_shared_prefix(prefix)
    rules = LogitsRules(repetition=torch.full((B,), 1e30, device=DEV))
    out = engine.generate(ids, n, new, rules=rules).cpu()
    logits = engine.prefill(ids, n, new)
    seen = [set(prefix.tolist()) | set(ids[b, : n[b]].tolist()) for b in range(B)]
    for step in range(new):
        z = logits.float().cpu()
        for b in range(B):
            said = torch.tensor(sorted(seen[b]))
            z[b, said] = torch.where(z[b, said] > 0, z[b, said] / 1e30, z[b, said] * 1e30)
            assert int(out[b, step]) == int(z[b].argmax()) and int(out[b, step]) not in seen[b]
            seen[b].add(int(out[b, step]))
        logits = engine.decode_step(out[:, step].to(DEV))
    engine.set_shared_prefix(None)
    assert engine.prefix_ids is None


@pytest.mark.parametrize("impl", ["tcgen05", "mma"])
@pytest.mark.parametrize("T,H,Hkv,D", [(3, 4, 2, 64), (64, 8, 2, 64), (65, 8, 8, 64), (300, 4, 1, 64), (5, 8, 2, 128), (200, 8, 2, 128)])
def test_attention_over_memory_as_an_unrounded_part(impl, T, H, Hkv, D):
    """Alone it joins to attention_fwd's own bits; beside another part nothing is rounded before the join."""
    from pdattention_b200.inference.shared_prefix import merge_attention_partials
    from pdattention_b200.ops import _ext

    torch.manual_seed(T)
    ext, B, w, n = _ext.require(), 3, Hkv * D, 70
    q = torch.randn(B, T, H * D, device=DEV).bfloat16()
    k, v = torch.randn(2, B, T, w, device=DEV).bfloat16()
    pool = torch.randn(500, 2 * w, device=DEV).bfloat16()
    idx = torch.randint(0, 500, (B, n), device=DEV, dtype=torch.int32)
    mem_len = torch.tensor([n, 0, 33], dtype=torch.int32, device=DEV)
    valid = torch.zeros(B, T, dtype=torch.uint8, device=DEV)  # the memory only
    args = (q, k, v, H, Hkv, D, pool[:, :w], pool[:, w:], idx, mem_len, valid, 1 / math.sqrt(D))
    ext.set_attention_impl(impl)
    try:
        o, ml = ext.attention_partials(*args)
        out, lse = ext.attention_fwd(*args)
    finally:
        ext.set_attention_impl("tcgen05")
    assert o.shape == (B * T, H, 1, D) and ml.shape == (B * T, H, 1, 2) and (ml[..., 1] == 1).all()
    alone, alone_lse = merge_attention_partials((o, ml), batch=B, return_lse=True)
    assert torch.equal(alone, out) and torch.equal(alone_lse, lse)
    assert (lse[1] == NEG_INF).all() and (out[1] == 0).all()
    o = o.view(B, T, H, D)
    seen = o[0::2]
    assert (seen.bfloat16().float() != seen).float().mean() > 0.9  # fp32 values
    keys = [pool[idx[b, : int(mem_len[b])].long()].double().view(-1, 2, Hkv, D).repeat_interleave(H // Hkv, 2) for b in (0, 2)]
    for b, kv in zip((0, 2), keys):
        x = q[b].double().view(T, H, D)
        s = torch.einsum("thd,nhd->htn", x, kv[:, 0]) / math.sqrt(D)
        p = torch.softmax(s, -1)
        want, mass = torch.einsum("htn,nhd->thd", p, kv[:, 1]), torch.einsum("htn,nhd->thd", p, kv[:, 1].abs())
        size = torch.einsum("thd,nhd->htn", x.abs(), kv[:, 0].abs()).amax() / math.sqrt(D)
        slack = D * 2.0 ** -24 * size + 2.0 ** -20 * (1 + size + torch.logsumexp(s, -1).abs().amax())
        # every weight half a step of bf16 and the score's error; no rounding of the result
        assert ((o[b].double() - want).abs() <= (half_step(torch.bfloat16) + 2 * slack) * mass).all()


def test_a_prefill_joins_its_memory_unrounded(monkeypatch):
    from test_serving_engine_gpu import setup

    from pdattention_b200.inference import llama_engine

    cfg, model, engine = setup(10)
    engine.build_memory(torch.randint(0, cfg.vocab_size, (12, 16)), torch.full((12,), 16, dtype=torch.int32))
    engine.set_namespace(torch.zeros(2, dtype=torch.int32), torch.full((2,), 12, dtype=torch.int32))
    engine.set_shared_prefix(torch.arange(30))
    parts = []
    join = llama_engine.merge_attention_partials
    monkeypatch.setattr(llama_engine, "merge_attention_partials", lambda a, b, **kw: (parts.append(b[0]), join(a, b, **kw))[1])
    engine.prefill(torch.randint(0, cfg.vocab_size, (2, 9)), torch.tensor([9, 4]), 2)
    assert len(parts) == cfg.num_hidden_layers
    for o in parts:
        assert o.dtype == torch.float32 and (o.bfloat16().float() != o).float().mean() > 0.9


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("tokens,heads,kv,dim,rot,interleaved", [(1, 8, 2, 64, 64, False), (77, 5, 1, 128, 64, True), (700, 4, 4, 80, 20, False),
                                                                 (9, 3, 3, 6, 2, True), (16, 0, 2, 64, 64, False)])
def test_rotary_cache_of_other_types(dtype, tokens, heads, kv, dim, rot, interleaved):
    from pdattention_b200.ops.rotary import rotary_cache, rotary_table

    torch.manual_seed(tokens)
    qkv = torch.randn(tokens, (heads + 2 * kv) * dim + 3, device=DEV).to(dtype)[:, : (heads + 2 * kv) * dim]
    pos = torch.randint(0, 1000, (tokens,), device=DEV)
    table = rotary_table(rot, 1000, interleaved=interleaved)
    rows = tokens + 20
    slots = torch.randperm(rows, device=DEV)[:tokens].int()
    if tokens > 2:
        slots[1], slots[2] = -1, rows  # not written
    kc, vc = torch.full((2, rows, kv * dim), 7.0, device=DEV, dtype=dtype)
    q = rotary_cache(qkv, heads, kv, dim, pos, table, kc, vc, slots)
    x = qkv.reshape(tokens, heads + 2 * kv, dim)
    want = rotate64(x, pos, table)
    if heads:
        rotary_close(q.view(tokens, heads, dim), want[:, :heads], x[:, :heads], rot)
    kept = (slots >= 0) & (slots < rows)
    at = slots[kept].long()
    rotary_close(kc[at].view(-1, kv, dim), want[kept, heads: heads + kv], x[kept, heads: heads + kv], rot)
    assert torch.equal(vc[at], x[kept, heads + kv:].flatten(1))
    rest = torch.ones(rows, dtype=torch.bool, device=DEV)
    rest[at] = False
    assert (kc[rest] == 7).all() and (vc[rest] == 7).all()


@pytest.mark.parametrize("B,T,P,H,Hkv,D", [(64, 1, 8192, 32, 8, 128), (16, 4, 4096, 32, 8, 128), (8, 5, 700, 12, 12, 64),
                                           (16, 16, 300, 4, 4, 128), (3, 60, 500, 8, 2, 64)])
@pytest.mark.parametrize("cap", [4096, 16384])
def test_capacities_far_above_the_lengths(B, T, P, H, Hkv, D, cap):
    """The rows of an engine's cache: room for many tokens more, whatever is in it."""
    from pdattention_b200.inference.shared_prefix import shared_prefix_attention

    torch.manual_seed(cap + B)
    w = Hkv * D
    q = (1.5 * torch.randn(B, T, H * D, device=DEV)).bfloat16()
    pk, pv = torch.randn(2, P, w, device=DEV).bfloat16()
    lengths = torch.randint(T, 150, (B,), device=DEV, dtype=torch.int32)
    k, v = torch.full((2, B, cap, w), float("nan"), device=DEV, dtype=torch.bfloat16)
    for b in range(B):
        n = int(lengths[b])
        k[b, :n], v[b, :n] = torch.randn(2, n, w, device=DEV).bfloat16()
    out, lse = shared_prefix_attention(q, pk, pv, k, v, lengths, H, Hkv, D, return_lse=True)
    prefix_close(out, lse, prefix64(q, pk, pv, k[:, :150], v[:, :150], lengths, None, H, Hkv, D, 1 / math.sqrt(D)), D)
