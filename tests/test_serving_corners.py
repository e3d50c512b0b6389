"""Corner calls of the serving operators that need no GPU."""

import itertools

import pytest
import torch

from pdattention_b200.ops import _ext

needs_ext = pytest.mark.skipif(not _ext.available(), reason="extension not built")


def views():
    """Tensors [..., heads, head_dim] whose leading dimensions have sizes of 1 with strides of any kind."""
    base = torch.arange(3 * 2 * 3 * 2 * 4).view(3, 2, 3, 2, 4)
    yield base[:, ::2]                                  # [3, 1, 3]: the middle stride is two rows
    yield base[:1].permute(1, 2, 0, 3, 4)               # [2, 3, 1]: the inner stride is the whole tensor
    yield base[:, :1, :1].transpose(0, 2)               # [1, 1, 3]
    yield base[:, :, ::3]                               # [3, 2, 1]
    yield base[:, 1]                                    # [3, 3]
    yield base.transpose(0, 1)                          # no one stride
    yield base[::2].transpose(0, 2)
    yield base[0, 0]
    yield base[:1, :1, :1]
    yield base[0, 0, 0]                                 # a single token without leading dimensions
    yield base[:, :1, 0, :1].expand(3, 4, 1, 4)         # broadcast: stride 0
    yield base[0, 0, :1].expand(5, 2, 4)
    for order in itertools.permutations(range(3)):
        for cut in itertools.product((slice(None), slice(0, 1), slice(None, None, 2)), repeat=3):
            yield base[cut].permute(*order, 3, 4)


@needs_ext
def test_token_stride_ignores_dimensions_of_one():
    found = 0
    for x in views():
        stride = _ext.require().token_stride(list(x.shape), list(x.stride()))
        tokens = x.shape[:-2].numel()
        first = x.reshape(tokens, *x.shape[-2:])[:, 0, 0]  # where each token begins, in elements of the base
        if stride >= 0:
            found += 1
            assert torch.equal(first, first[0] + stride * torch.arange(tokens)), (x.shape, x.stride())
        else:
            steps = first.diff()
            assert not (steps == steps[0]).all()  # there is none
    assert found > 50


def test_dynamic_scaling_matches_hugging_face_past_the_window():
    """A prompt behind the window, decode steps on its cache, and a prompt within the window."""
    import transformers

    from pdattention_b200.hf.convert import reference_from_hf
    from pdattention_b200.models.llama import hf_config, reference_step, tiny_llama
    from pdattention_b200.models.llama import PRALlamaReference

    source = PRALlamaReference(tiny_llama(max_position_embeddings=32)).eval()
    source.reset_parameters(seed=0, std=0.2)
    hcfg = hf_config(source.cfg)
    hcfg.rope_parameters = {"rope_type": "dynamic", "factor": 4.0, "rope_theta": source.cfg.rope_theta}
    hcfg._attn_implementation = "eager"
    fresh = lambda: transformers.LlamaForCausalLM(hcfg).eval()  # noqa: E731 (it keeps the longest length that it saw)
    hf = fresh()
    hf.load_state_dict(source.state_dict(), strict=False)
    ours = reference_from_hf(hf)
    assert ours.cfg.rope_scaling["rope_type"] == "dynamic"
    ids = torch.randint(0, source.cfg.vocab_size, (1, 103), generator=torch.Generator().manual_seed(1))
    # tolerance as in the comparison of the other scalings: the other side's angles are fp32
    close = lambda a, b: torch.allclose(a, b, atol=2e-3, rtol=1e-3)  # noqa: E731
    with torch.no_grad():
        within = hf(ids[:, :32]).logits
        assert close(ours(ids[:, :32]), within) and close(source(ids[:, :32]), within)  # not yet scaled
        out = hf(ids[:, :100], use_cache=True)
        assert close(ours(ids[:, :100]), out.logits)
        assert not torch.allclose(source(ids[:, :100]), out.logits, atol=2e-2, rtol=1e-2)
        cache = [[None, None] for _ in range(source.cfg.num_hidden_layers)]
        assert close(reference_step(ours, ids[0, :100], cache, None, None)[0], out.logits[0])
        for t in range(100, 103):
            out = hf(ids[:, t: t + 1], past_key_values=out.past_key_values, use_cache=True)
            assert close(reference_step(ours, ids[0, t: t + 1], cache, None, None)[0], out.logits[0])


def test_angles_of_sequences_of_several_lengths():
    from pdattention_b200.ops.rotary import rotary_angles, rotary_frequencies

    d = {"rope_type": "dynamic", "factor": 2.0, "original_max_position_embeddings": 100}
    pos = torch.arange(300).expand(3, 300)
    lengths = torch.tensor([300, 101, 60])
    got, one = rotary_angles(pos, 8, 10000.0, d, lengths[:, None])
    assert got.shape == (3, 300, 4) and one == 1.0
    for row, n in enumerate(lengths.tolist()):
        assert torch.allclose(got[row], torch.arange(300.0, dtype=torch.float64)[:, None] * rotary_frequencies(8, 10000.0, d, n)[0],
                              rtol=1e-13)
    steps, _ = rotary_angles(torch.arange(300), 8, 10000.0, d)  # each position the end of its sequence
    for p in (0, 50, 99, 100, 101, 299):
        assert torch.allclose(steps[p], p * rotary_frequencies(8, 10000.0, d, p + 1)[0], rtol=1e-13)
    for scaling in (None, {"type": "linear", "factor": 3.0}):  # lengths do not matter
        freq, _ = rotary_frequencies(8, 10000.0, scaling)
        assert torch.equal(rotary_angles(pos, 8, 10000.0, scaling, lengths[:, None])[0], pos.double()[..., None] * freq)
    assert torch.equal(rotary_angles(pos, 2, 10000.0, d, 300)[0][..., 0], pos.double())  # a single pair has no base


def test_history_behind_a_shared_prefix():
    from pdattention_b200.inference.logits import TokenHistory

    h = TokenHistory.start(torch.tensor([[5, 6], [7, 0]]), torch.tensor([2, 1]), 1, torch.tensor([8, 9, 8]))
    assert h.ids.tolist() == [[8, 9, 8, 5, 6, 0], [8, 9, 8, 7, 0, 0]]
    assert h.lengths.tolist() == h.prompt_lengths.tolist() == [5, 4]
    h.append(torch.tensor([1, 2]))
    assert h.ids.tolist() == [[8, 9, 8, 5, 6, 1], [8, 9, 8, 7, 2, 0]] and h.prompt_lengths.tolist() == [5, 4]
    alone = TokenHistory.start(torch.tensor([[5, 6]]), torch.tensor([2]), 1, torch.zeros(0, dtype=torch.long))
    assert alone.ids.tolist() == [[5, 6, 0]] and alone.lengths.tolist() == [2]


def prefix_engine(monkeypatch, rotary_cache):
    """An engine without kernels: ``set_shared_prefix`` runs, every layer leaves its input alone."""
    from types import SimpleNamespace

    from pdattention_b200.inference import llama_engine
    from pdattention_b200.models.llama import tiny_llama

    engine = llama_engine.PRALlamaEngine.__new__(llama_engine.PRALlamaEngine)
    cfg = tiny_llama(head_dim=64)
    engine.cfg, engine.device, engine.tp = cfg, torch.device("cpu"), None
    engine.heads, engine.kv_heads = cfg.num_attention_heads, cfg.num_key_value_heads
    engine.q_dim, engine.kv_dim = cfg.q_dim, cfg.kv_dim
    engine.prefix = engine.prefix_ids = engine.cache = None
    engine._rope_cache = {}
    engine.w = SimpleNamespace(layers=[SimpleNamespace(ln_in=None, qkv=None, qkv_bias=None, o=None)] * cfg.num_hidden_layers)
    monkeypatch.setattr(llama_engine, "rotary_cache", rotary_cache)
    monkeypatch.setattr(llama_engine, "shared_prefix_attention", lambda q, *a: q)
    engine._norm = engine._row_parallel = lambda x, *a, **kw: x
    engine._gemm = lambda x, *a, **kw: torch.zeros(x.shape[0], cfg.q_dim + 2 * cfg.kv_dim)
    engine._mlp = lambda lw, x: x
    engine._ln = lambda w: None
    engine._embed = lambda ids: torch.zeros(ids.numel(), cfg.hidden_size)
    return engine


def test_a_prefix_that_was_not_finished_is_none(monkeypatch):
    """An exception while the second chunk is encoded: the engine has no prefix, not half of one."""
    calls = []

    def rotary_cache(qkv, heads, kv_heads, head_dim, pos, table, k, v, rows):
        calls.append(int(rows[0]))
        if rows[0] >= 10:
            raise torch.OutOfMemoryError("no room")
        return qkv[:, : heads * head_dim]

    engine = prefix_engine(monkeypatch, rotary_cache)
    with pytest.raises(torch.OutOfMemoryError):
        engine.set_shared_prefix(torch.arange(25), chunk_tokens=10)
    assert max(calls) == 10 and engine.prefix is None and engine.prefix_ids is None and engine.prefix_tokens == 0
    engine.set_shared_prefix(torch.arange(9), chunk_tokens=10)
    assert engine.prefix_tokens == 9 and engine.prefix_ids.tolist() == list(range(9))


@pytest.mark.parametrize("chunk,room,size", [(10, 7, 7), (5, 7, 5), (4096, 0, 1)])
def test_prefix_chunks_fit_the_tensor_parallel_buffer(monkeypatch, chunk, room, size):
    """A chunk's row-parallel partials fit the peer buffer (one row at least)."""
    from types import SimpleNamespace

    chunks = []

    def rotary_cache(qkv, heads, kv_heads, head_dim, pos, table, k, v, rows):
        assert torch.equal(pos, rows)  # unscaled: a token's position is its row
        chunks.append(rows.tolist())
        return qkv[:, : heads * head_dim]

    engine = prefix_engine(monkeypatch, rotary_cache)
    engine.tp = SimpleNamespace(max_partial=room * engine.cfg.hidden_size + engine.cfg.hidden_size - 1)
    engine.set_shared_prefix(torch.arange(17), chunk_tokens=chunk)
    layers = engine.cfg.num_hidden_layers
    assert all(c == list(range(i // layers * size, min(17, (i // layers + 1) * size))) for i, c in enumerate(chunks))
    assert len(chunks) == -(-17 // size) * layers and engine.prefix_tokens == 17


@needs_ext
def test_derivatives_that_rotary_does_not_have_are_refused():
    import torch.autograd.forward_ad as fwad

    from pdattention_b200.ops.rotary import RotaryTable, rotary, rotary_table

    t = rotary_table(8, 4, device="cpu")
    q, pos = torch.randn(3, 2, 8), torch.zeros(3, dtype=torch.long)
    with fwad.dual_level():
        dual = fwad.make_dual(q, torch.ones_like(q))
        for args in ((dual, None), (q, dual), (dual.clone().requires_grad_(), None)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                rotary(*args, pos, t)
        with pytest.raises(RuntimeError, match="forward-mode"):
            rotary(q, None, pos, RotaryTable(fwad.make_dual(t.cos, t.cos), t.sin))
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            rotary(dual, None, pos, t)
    learned = RotaryTable(t.cos.clone().requires_grad_(), t.sin)
    for x in (q, q.clone().requires_grad_()):
        with pytest.raises(RuntimeError, match="gradients for its table"):
            rotary(x, None, pos, learned)
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA tensor"):  # without gradients any table serves
        rotary(q, None, pos, learned)


def test_choices_of_vocabulary_slices_are_joined():
    from pdattention_b200.inference.logits import join_choices

    nan, inf = float("nan"), float("inf")
    cases = [  # (value, id) of each slice: the choice over all of them
        ([(1.0, 3), (2.0, 40), (0.5, 99)], 40),
        ([(2.0, 3), (2.0, 40), (2.0, 99)], 3),        # ties: the lowest id
        ([(-inf, -1), (-5.0, 40), (-inf, -1)], 40),   # slices with nothing left
        ([(-inf, -1), (-inf, -1), (-inf, -1)], -1),
        ([(inf, 3), (nan, 40), (1.0, 99)], 40),       # NaN is larger than +inf
        ([(nan, 17), (inf, 40), (nan, 99)], 17),
        ([(inf, 3), (inf, 40), (-inf, -1)], 3),
        ([(-0.0, 7), (0.0, 40), (-1.0, 99)], 7),      # -0 counts as 0
        ([(-3.4e38, 7), (-inf, -1), (-3.4e38, 393215)], 7),
    ]
    values = torch.tensor([[v for v, _ in c] for c, _ in cases])
    tokens = torch.tensor([[t for _, t in c] for c, _ in cases])
    for ids in (tokens, tokens.float()):  # ids travel as fp32, exact under 2^24
        got = join_choices(values, ids)
        assert got.dtype == torch.int64 and got.tolist() == [t for _, t in cases]


def test_tensor_parallel_ranks_choose_alike(monkeypatch):
    """``_choose`` of two ranks (each with half of the columns) gives what one rank with all of them gives, and the
    same histories.  The kernel's place is taken by the operator's definition."""
    from types import SimpleNamespace

    from pdattention_b200.inference import llama_engine
    from pdattention_b200.inference.logits import LogitsRules, TokenHistory

    torch.manual_seed(0)
    B, V = 6, 32
    logits = torch.randn(B, V)
    logits[1, 20] = logits[1].amax() + 1
    logits[1, 5] = logits[1, 20]            # a tie across the ranks
    logits[2] = float("-inf")               # nothing left
    logits[3, 3], logits[3, 30] = float("inf"), float("nan")
    logits[4, 16:] = float("-inf")          # one rank with nothing left

    def choose(local, rules, history, vocab_start=0, append=False):
        key = torch.where(local.isnan(), float("inf"), local)
        key = torch.where(local.isnan().any(1, keepdim=True) & ~local.isnan(), float("-inf"), key)
        value, at = key.max(1)
        value = local.gather(1, at[:, None])[:, 0]
        token = torch.where(value == float("-inf"), -1, at + vocab_start)
        if append:
            history.append(token)
        return token, value

    monkeypatch.setattr(llama_engine, "choose_tokens", choose)

    def engine(start, tp, size):
        e = llama_engine.PRALlamaEngine.__new__(llama_engine.PRALlamaEngine)
        e.vocab_start, e.tp, e.tp_size = start, tp, size
        return e

    fresh = lambda: TokenHistory(torch.zeros(B, 3, dtype=torch.int32), torch.tensor([0, 1, 2, 0, 3, 0], dtype=torch.int32))  # noqa: E731
    rules, want_history = LogitsRules(), fresh()
    want = engine(0, None, 1)._choose(logits, rules, want_history)
    assert want[1:5].tolist() == [5, -1, 30, int(logits[4].argmax())]
    pairs = []
    for half in range(2):
        part = logits[:, half * 16: half * 16 + 16]
        token, value = choose(part, rules, None, vocab_start=half * 16)
        pairs.append(torch.stack([value, token.float()], 1))
    for half in range(2):
        sent = []
        tp = SimpleNamespace(gather_small=lambda x: (sent.append(x), torch.cat(pairs, 1))[1])
        history = fresh()
        got = engine(half * 16, tp, 2)._choose(logits[:, half * 16: half * 16 + 16], rules, history)
        assert torch.equal(got, want) and got.dtype == want.dtype
        assert torch.equal(sent[0].nan_to_num(nan=7.0), pairs[half].nan_to_num(nan=7.0))
        assert torch.equal(history.ids, want_history.ids) and torch.equal(history.lengths, want_history.lengths)


def test_rules_and_histories_that_a_step_would_ignore_are_refused():
    from pdattention_b200.inference.llama_engine import PRALlamaEngine
    from pdattention_b200.inference.logits import LogitsRules, TokenHistory

    engine = PRALlamaEngine.__new__(PRALlamaEngine)
    history = TokenHistory(torch.zeros(1, 3, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError, match="sample=True"):
        engine.decode_step(torch.zeros(1, dtype=torch.long), rules=LogitsRules())
    with pytest.raises(ValueError, match="history without rules"):
        engine.decode_step(torch.zeros(1, dtype=torch.long), sample=True, history=history)
    with pytest.raises(ValueError, match="sample=True"):
        engine.capture_decode(rules=LogitsRules())


def test_rows_of_nothing_but_the_prefix_are_refused():
    from pdattention_b200.inference.llama_engine import PRALlamaEngine
    from pdattention_b200.models.llama import tiny_llama

    engine = PRALlamaEngine.__new__(PRALlamaEngine)
    engine.cfg, engine.prefix = tiny_llama(), torch.zeros(2, 5, 8)
    for ids, n in ((torch.zeros(3, 4), [4, 0, 1]), (torch.zeros(1, 0), [0]), (torch.zeros(2, 1), [1, -1])):
        with pytest.raises(ValueError, match="token of its own"):
            engine.prefill(ids.long(), torch.tensor(n), 4)


def test_the_window_of_dynamic_scaling_to_and_from_hugging_face():
    """Hugging Face has no original window for it: ``max_position_embeddings`` is the window."""
    import transformers

    from pdattention_b200.hf.convert import config_from_hf
    from pdattention_b200.models.llama import PRALlamaReference, hf_config, tiny_llama

    hcfg = transformers.LlamaConfig(hidden_size=64, num_attention_heads=4, head_dim=16, max_position_embeddings=128, rope_parameters={
        "rope_type": "dynamic", "factor": 4.0, "rope_theta": 1e4, "original_max_position_embeddings": 32})
    assert config_from_hf(hcfg).rope_scaling["original_max_position_embeddings"] == 128
    cfg = tiny_llama(max_position_embeddings=128, rope_scaling={"rope_type": "dynamic", "factor": 4.0,
                                                                "original_max_position_embeddings": 32})
    ours = PRALlamaReference(cfg).eval()
    ours.reset_parameters(seed=0, std=0.2)
    hcfg = hf_config(cfg)
    hcfg._attn_implementation = "eager"
    hf = transformers.LlamaForCausalLM(hcfg).eval()
    hf.load_state_dict(ours.state_dict(), strict=False)
    ids = torch.randint(0, cfg.vocab_size, (1, 100), generator=torch.Generator().manual_seed(1))
    with torch.no_grad():  # tolerance as above
        assert torch.allclose(ours(ids), hf(ids).logits, atol=2e-3, rtol=1e-3)
    assert cfg.rope_scaling["original_max_position_embeddings"] == 32
    assert config_from_hf(hcfg).rope_scaling["original_max_position_embeddings"] == 32
