"""The tree operators as a decoding loop uses them: m5_forward_tree against
m5_forward, and tree_speculative_generate_step against the main model's plain
greedy decode.

A node's logits come from the same weights and the same visible keys as those
of a plain call on its path, through another attention kernel (fp32 scores
where the plain one rounds them to bf16) and, above 15 rows, the GEMM instead of the
GEMV; the bound is the one the plain calls' chunked prefill is held to, 0.05
max-abs.  Streams are compared up to the first step whose top-2 gap in the plain
run is below 0.05, where either token is right."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

MAIN = dict(model_type="qwen3", hidden_size=512, num_hidden_layers=3, num_attention_heads=8, num_key_value_heads=2,
            head_dim=128, intermediate_size=1024, vocab_size=4096, tie_word_embeddings=False,
            max_position_embeddings=40960, rms_norm_eps=1e-6, rope_theta=1e6)
DRAFT = dict(MAIN, hidden_size=256, num_hidden_layers=2, num_attention_heads=4, intermediate_size=512)


def _model(cfg, seed):
    from myinfer_b200.model import Model, ModelArgs, upload_weights
    from oracle import model as om
    return Model(ModelArgs.from_dict(cfg), upload_weights(om.generate_weights(om.Config.from_dict(cfg), seed), "cuda"),
                 "cuda", max_tokens=64)


def _prefilled(model, prompt, kv_bits):
    from myinfer_b200.attention import safe_maybe_quantize_kv_cache
    from myinfer_b200.cache import make_prompt_cache
    cache = make_prompt_cache(model)
    model.forward(torch.tensor(prompt, dtype=torch.int32).cuda(), cache)
    safe_maybe_quantize_kv_cache(cache, 0, 64, kv_bits)
    for c in cache:
        c.reserve(len(prompt) + 80)
    return cache


@pytest.mark.parametrize("kv_bits", [None, 4, 8])
@pytest.mark.parametrize("split", [0, 3])
def test_forward_tree_matches_paths(kv_bits, split):
    """Every node's logits equal a plain forward of its path, whether the tree comes in one call or two."""
    from myinfer_b200 import _lib
    from myinfer_b200.tree import tree_plan
    model = _model(MAIN, 5)
    rng = np.random.default_rng(3)
    prompt = rng.integers(0, MAIN["vocab_size"], 37).tolist()
    par = [-1, 0, 0, 1, 1, 2, 4, 6, 6]
    tok = rng.integers(0, MAIN["vocab_size"], len(par)).astype(np.int32)
    T, V = len(par), MAIN["vocab_size"]
    parents = torch.tensor([par], dtype=torch.int32).cuda()
    anc, depth = tree_plan(parents)
    cache = _prefilled(model, prompt, kv_bits)
    toks = torch.from_numpy(tok).cuda()
    logits = torch.empty(T, V, dtype=torch.bfloat16, device="cuda")
    for a, b in ([(0, split), (split, T)] if split else [(0, T)]):
        model.forward_tree(toks[a:b], cache, depth[0, a:b], anc[0, a:b], a, _lib.M5_LOGITS_ALL, logits[a:b])
    assert cache.offset == len(prompt)
    _lib.device_check()
    for i in range(T):
        path, j = [], i
        while j >= 0:
            path.append(int(tok[j]))
            j = par[j]
        plain = _prefilled(model, prompt, kv_bits)
        want = torch.empty(V, dtype=torch.bfloat16, device="cuda")
        model.forward(torch.tensor(path[::-1], dtype=torch.int32).cuda(), plain, _lib.M5_LOGITS_LAST, want)
        err = (logits[i].float() - want.float()).abs().max().item()
        assert err <= 0.05, (i, err)


def _plain(model, prompt, n, kv_bits):
    from myinfer_b200.generate import generate_step
    out = list(generate_step(prompt, model, n, prefill_step_size=16, kv_bits=kv_bits, quantized_kv_start=0,
                             return_logits=True))
    return [t for t, _ in out], [l.float().cpu() for _, l in out]


def _agree(spec, plain, logits):
    for i, (a, b) in enumerate(zip(spec, plain)):
        if a != b:
            top2 = logits[i].topk(2).values
            assert (top2[0] - top2[1]).item() < 0.05, (i, a, b)
            return


@pytest.mark.parametrize("widths,kv_bits", [((1,), 8), ((1, 1, 1), 4), ((3, 2, 1), 8), ((4, 3, 2), None), ((7, 3, 1), 4)])
def test_tree_speculation_equals_greedy(widths, kv_bits):
    from myinfer_b200.generate import tree_speculative_generate_step
    main, draft = _model(MAIN, 31), _model(DRAFT, 32)
    prompt = np.random.default_rng(len(widths)).integers(0, MAIN["vocab_size"], 30).tolist()
    n = 24
    plain, logits = _plain(main, prompt, n, kv_bits)
    got = list(tree_speculative_generate_step(prompt, main, draft, widths, n, prefill_step_size=16, kv_bits=kv_bits,
                                              quantized_kv_start=0))
    assert len(got) == n
    _agree([t for t, _ in got], plain, logits)


def test_self_draft_accepts_whole_paths():
    """The main model as its own draft: its first choice at every node is the main model's, so all but each
    round's last token come from the draft (less a proposal lost at a near-tie of the two calls)."""
    from myinfer_b200.cache import make_prompt_cache
    from myinfer_b200.generate import tree_speculative_generate_step
    main = _model(MAIN, 33)
    prompt = list(range(5, 40))
    n = 20
    plain, logits = _plain(main, prompt, n, 8)
    mc, dc = make_prompt_cache(main), make_prompt_cache(main)
    got = list(tree_speculative_generate_step(prompt, main, main, (2, 2, 1, 1), n, prompt_cache=mc, draft_cache=dc,
                                              prefill_step_size=16, kv_bits=8, quantized_kv_start=0))
    _agree([t for t, _ in got], plain, logits)
    assert sum(d for _, d in got) >= n - n // 5 - 3
    assert mc.offset == dc.offset
    # what the caches keep is the path: a plain call goes on from it as from a fresh prefill of the same tokens
    ctx = prompt + [t for t, _ in got]
    keep = ctx[:mc.offset]
    fresh = _prefilled(main, keep, 8)
    from myinfer_b200 import _lib
    nxt = torch.tensor([ctx[mc.offset] if mc.offset < len(ctx) else 1], dtype=torch.int32).cuda()
    a, b = (torch.empty(MAIN["vocab_size"], dtype=torch.bfloat16, device="cuda") for _ in range(2))
    main.forward(nxt, mc, _lib.M5_LOGITS_LAST, a)
    main.forward(nxt, fresh, _lib.M5_LOGITS_LAST, b)
    cos = torch.nn.functional.cosine_similarity(a.float(), b.float(), dim=0).item()
    assert cos >= 0.999, cos


def test_constrained_speculation():
    """A grammar that allows one token in five, a bias and penalties: every token obeys the mask, and widths do not
    change the stream (up to a near-tie of the processed logits, which is not known here: the first tokens)."""
    from myinfer_b200.generate import tree_speculative_generate_step
    main, draft = _model(MAIN, 35), _model(DRAFT, 36)
    V = MAIN["vocab_size"]
    allowed = np.zeros(V, bool)
    allowed[::5] = True
    words = np.packbits(allowed, bitorder="little").view(np.int32)

    def grammar(tokens, nodes, parents):
        return torch.from_numpy(np.tile(words, (len(nodes), 1))).cuda()
    kw = dict(max_tokens=16, penalties=(1.3, 0.2, 0.1), logit_bias={5: 1.0, 15: 0.5, 7: 50.0}, grammar=grammar,
              prefill_step_size=16, kv_bits=8, quantized_kv_start=0)
    prompt = list(range(100, 130))
    wide = [t for t, _ in tree_speculative_generate_step(prompt, main, draft, (3, 2), **kw)]
    thin = [t for t, _ in tree_speculative_generate_step(prompt, main, draft, (1,), **kw)]
    assert len(wide) == len(thin) == 16 and all(t % 5 == 0 for t in wide + thin)
    assert wide[:2] == thin[:2]
    none = list(tree_speculative_generate_step(prompt, main, draft, (2,), max_tokens=4, prefill_step_size=16,
                                               grammar=lambda *_: torch.zeros(3, V // 32, dtype=torch.int32, device="cuda")))
    assert none == []  # the grammar ends at once


def test_sampled_speculation_and_refusals():
    from myinfer_b200.generate import tree_speculative_generate_step
    from myinfer_b200.sample import DeviceSampler, make_logits_processors, make_sampler
    main, draft = _model(MAIN, 37), _model(DRAFT, 38)
    prompt = [1, 2, 3, 4]
    got = list(tree_speculative_generate_step(prompt, main, draft, (2, 1), 12, sampler=make_sampler(0.8, top_p=0.9, seed=4)))
    assert len(got) == 12 and all(0 <= t < MAIN["vocab_size"] for t, _ in got)
    for kw, text in ((dict(tree_widths=(64,)), "64 nodes"), (dict(tree_widths=(0,)), "positive"),
                     (dict(sampler=lambda x: x), "DeviceSampler"),
                     (dict(sampler=DeviceSampler(0.5, processors=make_logits_processors(1.1))), "penalties")):
        with pytest.raises(ValueError, match=text):
            next(tree_speculative_generate_step(prompt, main, draft, **kw))
    from myinfer_b200.cache import make_prompt_cache
    cache = make_prompt_cache(main, 64)
    t = torch.zeros(65, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        main.forward_tree(t[:2], cache, t[:2], t[:2])
    from myinfer_b200._lib import M5CudaError
    with pytest.raises(M5CudaError, match="64 nodes"):
        main.forward_tree(t, cache, t, torch.zeros(65, dtype=torch.int64, device="cuda"))


def test_stream_generate_tree():
    from myinfer_b200.generate import stream_generate

    class Tok:
        eos_token_ids = []

        def decode(self, ids):
            return " ".join(str(i) for i in ids)
    main, draft = _model(MAIN, 31), _model(DRAFT, 32)
    out = list(stream_generate(main, Tok(), [3, 1, 4, 1, 5], 10, draft_model=draft, tree_widths=(2, 2), kv_bits=8,
                               prefill_step_size=16))
    assert len(out) == 10 and out[-1].finish_reason == "length"


def _rows(cache, n):
    """K and V of the first n rows, fp32 [layers, 2, Hkv, n, D]."""
    from myinfer_b200 import ops
    return torch.stack([torch.stack([(ops.dequantize(*t, 64, c.bits) if c.bits else t)[0, :, :n].float()
                                     for t in (c.keys, c.values)]) for c in cache])


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("cached,prompt_len,start", [(0, 30, 40), (0, 1, 0), (20, 1, 0)],
                         ids=["threshold_crossed", "one_token", "given_bf16_cache"])
def test_rows_survive_quantization(cached, prompt_len, start, bits):
    """The cache turns to 8/4 bits while the loop runs: the committed rows are those of a fresh prefill of the same
    tokens.  Both were rounded to codes, at most a step (a fifteenth of a group's range, 0.3 of a row's
    size) and what the layers below make of it apart: less than half of a row's size; a lost row is off by all of it."""
    from myinfer_b200.cache import KVCache, make_prompt_cache
    from myinfer_b200.generate import tree_speculative_generate_step
    main, draft = _model(MAIN, 41), _model(DRAFT, 42)
    rng = np.random.default_rng(prompt_len)
    before = rng.integers(0, MAIN["vocab_size"], cached).tolist()
    prompt = rng.integers(0, MAIN["vocab_size"], prompt_len).tolist()
    caches = []
    for m in (main, draft):
        caches.append(_prefilled(m, before, None) if cached else make_prompt_cache(m))
    n = 20
    got = list(tree_speculative_generate_step(prompt, main, draft, (2, 2, 1), n, prompt_cache=caches[0],
                                              draft_cache=caches[1], prefill_step_size=16, kv_bits=bits,
                                              quantized_kv_start=start))
    assert len(got) == n
    ctx = before + prompt + [t for t, _ in got]
    for m, cache in zip((main, draft), caches):
        assert not any(type(c) is KVCache for c in cache)
        rows = min(cache.offset, len(ctx))
        assert rows >= len(ctx) - 1
        have, want = _rows(cache, rows), _rows(_prefilled(m, ctx[:rows], bits), rows)
        err = (have - want).norm(dim=-1) / want.norm(dim=-1)
        assert err.max().item() < 0.5, (err > 0.5).nonzero()[:5].tolist()


def test_prompt_and_decode_times():
    """The prompt's rate is of its own time, and the generation's does not hold it."""
    from myinfer_b200.generate import stream_generate, tree_speculative_generate_step

    class Tok:
        eos_token_ids = []

        def decode(self, ids):
            return " ".join(str(i) for i in ids)
    main, draft = _model(MAIN, 31), _model(DRAFT, 32)
    stats = {}
    list(tree_speculative_generate_step(list(range(200)), main, draft, (2,), 4, stats=stats, prefill_step_size=16))
    assert stats["prompt_tokens"] == 200 and stats["prompt_time"] > 0 and stats["decode_time"] > 0
    last = list(stream_generate(main, Tok(), list(range(200)), 4, draft_model=draft, tree_widths=(2,), prefill_step_size=16))[-1]
    assert 0 < last.prompt_tps < 1e7  # 200 tokens in 26 calls of the two models: not in 20 us


def test_context_of_a_reused_cache():
    """Tokens that a given cache holds count for the penalties and reach the grammar, once the caller names them."""
    from myinfer_b200.generate import tree_speculative_generate_step
    main, draft = _model(MAIN, 43), _model(DRAFT, 44)
    V, before, prompt = MAIN["vocab_size"], [7, 8, 9, 7, 50], [11, 12]
    seen = []

    def grammar(tokens, nodes, parents):
        seen.append(list(tokens))
        return torch.full((len(nodes), V // 32), -1, dtype=torch.int32, device="cuda")

    def run(**kw):
        caches = [_prefilled(m, before, None) for m in (main, draft)]
        seen.clear()
        return [t for t, _ in tree_speculative_generate_step(
            prompt, main, draft, (2, 1), 6, penalties=(1.0, 1000.0, 0.0), logit_bias={7: 50.0, 1500: 40.0}, grammar=grammar,
            prompt_cache=caches[0], draft_cache=caches[1], **kw)]
    got = run(context_tokens=before)
    # token 7 has been said: 1000 less; 1500 is said once
    assert 7 not in got and got[0] == 1500 and 1500 not in got[1:]
    assert seen[0] == before + prompt[:-1]
    assert run()[0] == 7 and seen[0] == prompt[:-1]  # without them only the prompt counts
    for bad in (before[:-1], before + [1], [7, 8, 9, 7, V], [7, 8, 9, 7, -1]):
        with pytest.raises(ValueError, match="context_tokens"):
            run(context_tokens=bad)


def test_forward_tree_refusals():
    """A logits buffer that the call would write past, or of another type, and a cache of several sequences."""
    from myinfer_b200 import _lib
    from myinfer_b200.cache import KVCache, PromptCache, make_prompt_cache
    from myinfer_b200.tree import tree_plan
    main = _model(MAIN, 37)
    V = MAIN["vocab_size"]
    anc, depth = tree_plan(torch.tensor([[-1, 0, 0]], dtype=torch.int32).cuda())
    tok = torch.zeros(3, dtype=torch.int32, device="cuda")
    cache = make_prompt_cache(main, 64)
    new = lambda *s, **kw: torch.empty(*s, **{**dict(dtype=torch.bfloat16, device="cuda"), **kw})  # noqa: E731
    for mode, lg in ((_lib.M5_LOGITS_ALL, new(2, V)), (_lib.M5_LOGITS_ALL, new(3, V, dtype=torch.float32)),
                     (_lib.M5_LOGITS_ALL, new(3, V, device="cpu")), (_lib.M5_LOGITS_ALL, new(3, 2 * V)[:, :V]),
                     (_lib.M5_LOGITS_ALL, None), (_lib.M5_LOGITS_LAST, new(V - 1))):
        with pytest.raises(ValueError, match="logits"):
            main.forward_tree(tok, cache, depth[0], anc[0], 0, mode, lg)
    batch = PromptCache([KVCache(main.n_kv_heads_local, 128, "cuda", 64, batch=2) for _ in range(3)], "cuda")
    with pytest.raises(ValueError, match="one sequence"):
        main.forward_tree(tok, batch, depth[0], anc[0])
    main.forward_tree(tok, cache, depth[0], anc[0], 0, _lib.M5_LOGITS_LAST, new(V))
    main.forward_tree(tok, cache, depth[0], anc[0], 0, _lib.M5_LOGITS_ALL, new(5, V))
    _lib.device_check()


def test_processors_of_the_other_loops():
    """What a caller of every loop passes, an empty list of logits processors, is taken; penalties over a window are
    refused with the reason."""
    from myinfer_b200.generate import stream_generate
    from myinfer_b200.sample import make_logits_processors

    class Tok:
        eos_token_ids = []

        def decode(self, ids):
            return " ".join(str(i) for i in ids)
    main, draft = _model(MAIN, 31), _model(DRAFT, 32)
    kw = dict(max_tokens=4, draft_model=draft, tree_widths=(2,), prefill_step_size=16)
    want = [r.token for r in stream_generate(main, Tok(), [3, 1, 4], **kw)]
    for none in (None, make_logits_processors()):
        assert [r.token for r in stream_generate(main, Tok(), [3, 1, 4], logits_processors=none, **kw)] == want
    with pytest.raises(ValueError, match="penalties"):
        next(stream_generate(main, Tok(), [3, 1, 4], logits_processors=make_logits_processors(1.2), **kw))
