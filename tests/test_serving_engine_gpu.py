"""The Llama engine with a shared prefix, scaled rotary positions and logits rules, against the fp32 oracle.

Logits are compared by cosine with the bounds of the engine's other tests (bf16 weights and
activations through two layers): 0.995 after a prefill, 0.99 after decode steps.
"""

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

LLAMA3 = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
          "original_max_position_embeddings": 64}


@pytest.fixture(scope="module", autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.skip("CUDA device required")


def setup(seed=0, head_dim=64, heads=4, kv_heads=2, **kw):
    from pdattention_b200.inference.llama_engine import LlamaWeights, PRALlamaEngine
    from pdattention_b200.models.llama import PRALlamaReference, tiny_llama

    torch.manual_seed(seed)
    cfg = tiny_llama(**{**dict(head_dim=head_dim, hidden_size=128, num_attention_heads=heads,
                               num_key_value_heads=kv_heads, chunk_tokens=16, top_k_chunks=3), **kw})
    model = PRALlamaReference(cfg).eval()
    model.reset_parameters(seed=seed, std=0.08)
    return cfg, model, PRALlamaEngine(LlamaWeights.from_reference(model, "cuda"), "cuda", decode_split_keys=64)


def close(got, want, bound):
    cos = F.cosine_similarity(got.float().cpu(), want, dim=-1)
    assert (cos > bound).all(), cos


@pytest.mark.parametrize("head_dim,scaling", [(64, LLAMA3), (128, {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32}),
                                              (64, {"type": "linear", "factor": 2.0})])
def test_scaled_positions(head_dim, scaling):
    from pdattention_b200.models.llama import reference_step

    cfg, model, engine = setup(1, head_dim, rope_scaling=scaling)
    ids, n = torch.randint(0, cfg.vocab_size, (2, 90)), torch.tensor([90, 41])
    logits = engine.prefill(ids, n, 3)
    caches = [[[None, None] for _ in range(cfg.num_hidden_layers)] for _ in range(2)]
    for b in range(2):
        close(logits[b], reference_step(model, ids[b, : n[b]], caches[b], None, None)[0][-1], 0.995)
    for _ in range(2):
        tok = torch.randint(0, cfg.vocab_size, (2,))
        got = engine.decode_step(tok)
        for b in range(2):
            close(got[b], reference_step(model, tok[b: b + 1], caches[b], None, None)[0][-1], 0.99)


@pytest.mark.parametrize("memory,overlap", [(False, True), (True, True), (True, False)])
@pytest.mark.parametrize("P,chunk,head_dim,B", [(1, 4096, 64, 2), (200, 64, 64, 3), (150, 150, 128, 70)])
def test_shared_prefix_matches_oracle(P, chunk, head_dim, B, memory, overlap):
    from pdattention_b200.models.llama import reference_step

    cfg, model, engine = setup(2, head_dim)
    engine.overlap_routing = overlap
    prefix = torch.randint(0, cfg.vocab_size, (P,))
    ref_mem = ns = None
    if memory:
        chunks, lengths = torch.randint(0, cfg.vocab_size, (12, 16)), torch.tensor([16, 16, 11, 16, 16, 9, 16, 16, 16, 13, 16, 16])
        engine.build_memory(chunks, lengths)
        engine.set_namespace(torch.arange(B) % 3, torch.full((B,), 12))
        ref_mem = model.encode_chunks(chunks, lengths)
    engine.set_shared_prefix(prefix, chunk_tokens=chunk)
    T = 20
    ids, n = torch.randint(0, cfg.vocab_size, (B, T)), torch.randint(1, T + 1, (B,))
    logits = engine.prefill(ids, n, 4, row_batch=None if B < 10 else 32)
    check = range(B) if B < 10 else (0, 31, 32, 69)
    caches = {}
    for b in check:
        caches[b] = [[None, None] for _ in range(cfg.num_hidden_layers)]
        reference_step(model, prefix, caches[b], None, None)  # prefix tokens read no memory
        ns = list(range(b % 3, 12)) if memory else None
        close(logits[b], reference_step(model, ids[b, : n[b]], caches[b], ref_mem, ns)[0][-1], 0.995)
    for _ in range(2):
        tok = torch.randint(0, cfg.vocab_size, (B,))
        got = engine.decode_step(tok)
        for b in check:
            ns = list(range(b % 3, 12)) if memory else None
            close(got[b], reference_step(model, tok[b: b + 1], caches[b], ref_mem, ns)[0][-1], 0.99)
    engine.set_shared_prefix(None)  # and the rows stand alone again
    alone = engine.prefill(ids, n, 1, row_batch=None if B < 10 else 32)
    for b in list(check)[:2]:
        cache = [[None, None] for _ in range(cfg.num_hidden_layers)]
        ns = list(range(b % 3, 12)) if memory else None
        close(alone[b], reference_step(model, ids[b, : n[b]], cache, ref_mem, ns)[0][-1], 0.995)


def test_generate_with_rules():
    from pdattention_b200.inference.logits import LogitsRules

    cfg, model, engine = setup(3)
    B, T, new, V = 3, 10, 12, cfg.vocab_size
    ids, n = torch.randint(0, V, (B, T)), torch.tensor([10, 4, 7])
    allowed = torch.zeros(B, V, dtype=torch.bool)
    allowed[0, 5:40] = True
    allowed[1] = True
    allowed[2, 77] = True
    words = (allowed.view(B, -1, 32).long() << torch.arange(32)).sum(-1).to(torch.int32).cuda()
    rules = LogitsRules(presence=torch.full((B,), 1e4, device="cuda"), mask=words)
    rules.presence[2] = 0
    out = engine.generate(ids, n, new, rules=rules).cpu()
    assert len(set(out[0].tolist())) == new and all(5 <= t < 40 for t in out[0].tolist())
    assert len(set(out[1].tolist())) == new  # a token said once is not said again
    assert out[2].tolist() == [77] * new
    # teacher-forced: every token is the best of what the engine's own logits leave
    logits = engine.prefill(ids, n, new)
    said = [set() for _ in range(B)]
    for step in range(new):
        z = logits.float().cpu().masked_fill(~allowed, float("-inf"))
        for b in range(2):
            z[b, list(said[b])] -= 1e4
            assert int(z[b].argmax()) == int(out[b, step])
            said[b].add(int(out[b, step]))
        logits = engine.decode_step(out[:, step].cuda())
    rules.mask[0] = 0  # a row with nothing left
    out = engine.generate(ids, n, 3, rules=rules).cpu()
    assert out[0].tolist() == [-1, -1, -1] and out[2].tolist() == [77] * 3


def test_prefix_scaling_and_rules_in_a_captured_step():
    """All of them in one decode step, eager and replayed: the same tokens."""
    from pdattention_b200.inference.logits import LogitsRules, TokenHistory, choose_tokens

    outs = []
    for graphed in (False, True):
        cfg, model, engine = setup(4, rope_scaling=LLAMA3)
        engine.build_memory(torch.randint(0, cfg.vocab_size, (12, 16)), torch.full((12,), 16, dtype=torch.int32))
        engine.set_namespace(torch.zeros(2, dtype=torch.int32), torch.full((2,), 12, dtype=torch.int32))
        engine.set_shared_prefix(torch.randint(0, cfg.vocab_size, (100,)))
        ids, n, new = torch.randint(0, cfg.vocab_size, (2, 12)), torch.tensor([12, 9]), 8
        rules = LogitsRules(repetition=torch.tensor([1.3, 1.1], device="cuda"), frequency=torch.full((2,), 0.2, device="cuda"),
                            bias_ids=torch.tensor([[3, 9], [9, -1]], device="cuda", dtype=torch.int32),
                            bias_values=torch.tensor([[-2.0, 1.0], [0.5, 9.0]], device="cuda"))
        history = TokenHistory.start(ids.cuda(), n, new)
        tok = choose_tokens(engine.prefill(ids, n, new), rules, history, append=True)[0]
        seq = [tok.clone()]
        tok = engine.decode_step(tok, sample=True, rules=rules, history=history)
        seq.append(tok.clone())
        if graphed:
            before = history.lengths.clone(), history.ids.clone(), engine.cache_len.clone()
            engine.capture_decode(sample=True, rules=rules, history=history)
            assert all(torch.equal(a, b) for a, b in zip(before, (history.lengths, history.ids, engine.cache_len)))
        for _ in range(new - 2):
            tok = engine.decode_step_graphed(tok) if graphed else engine.decode_step(tok, sample=True, rules=rules, history=history)
            seq.append(tok.clone())
        assert history.lengths.tolist() == [12 + new, 9 + new] and engine.cache_len.tolist() == [12 + new - 1, 9 + new - 1]
        outs.append(torch.stack(seq))
        engine.release_graph()
    assert torch.equal(outs[0], outs[1])


def test_refused_prefixes():
    cfg, model, engine = setup(5, head_dim=32)
    with pytest.raises(ValueError, match="head dim"):
        engine.set_shared_prefix(torch.arange(5))
    cfg, model, engine = setup(5)
    with pytest.raises(ValueError, match="one row"):
        engine.set_shared_prefix(torch.zeros(2, 5, dtype=torch.long))
    with pytest.raises(ValueError, match="scaling"):
        setup(5, rope_scaling={"rope_type": "other"})
