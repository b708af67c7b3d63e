"""The framework's own paths in four bits: the cache calls of the attention
module, the Llama host with 4-bit matrices, the engine with its handoff, its
scores, and the two-rank pilot.  Their 16-bit forms over the rounded values,
and the 64-bit oracle, say what has to come out."""
import json

import numpy as np
import pytest
import torch

from hexgen2_amd import fp4, llama, mha
from hexgen2_amd.engine import Engine
from hexgen2_amd.generation import InferenceParams
from hexgen2_amd.logprobs import token_logprobs
from oracle import mx_oracle as oracle
from tests.test_gpu_engine import GOLDEN, run_split
from tests.test_gpu_mx import DTYPES, attend_tolerance, randn, wide
from tests.test_gpu_pilot import launch

pytestmark = pytest.mark.gpu

MODEL = GOLDEN / "fixture_seed17"  # 2 layers, hidden 128, 4 heads of 32 on 2 KV heads, vocab 128
PROMPT = [5, 17, 90, 3, 44, 121, 8, 8, 63]

# Two orders of the same fp32 sums, at most 256 terms each: 256 * 2^-24 of the
# sum of magnitudes, about ten such sums one after the other (5 products a
# layer), their values a few times smaller than the sums of magnitudes:
# 10 * 8 * 256 * 2^-24 = 1.2e-3 of the largest logit.
LOGITS = 1.3e-3


def close(a, b):
    a, b = wide(a), wide(b)
    return np.abs(a - b).max() <= LOGITS * np.abs(b).max()


# ------------------------------------------------------------ cache calls ---


@pytest.mark.parametrize("dtype", DTYPES)
def test_cache_calls_attend_what_they_store(device, dtype):
    hq, h, d, b = 8, 2, 64, 3
    params = InferenceParams(60, max_batch_size=5, batch_size_offset=1, kv_bits=4)
    kv = randn((b, 48, 2, h, d), 1, dtype, device)
    q = randn((b, 48, hq, d), 2, dtype, device, 2.0)
    attn = mha.FlashCrossAttention(causal=True)
    stored = oracle.rounded(wide(kv))
    # the prompt gets its own rows back, to attend them as they were computed
    prompt = kv[:, :40]
    assert torch.equal(mha._update_kv_cache(prompt, params, 0), prompt)
    cache = params.key_value_memory_dict[0]
    assert cache.dtype == torch.uint8 and cache.shape == (5, 60, fp4.row_bytes(h, d))
    assert np.array_equal(wide(fp4.load_kv(cache[1:4], 40, h, d, torch.float32)), stored[:, :40])
    # a chunk, causal over the cache
    params.sequence_len_offset = 40
    view = mha._update_kv_cache(kv[:, 40:45], params, 0)
    got = attn(q[:, 40:45], view)
    want = oracle.attend(wide(q[:, 40:45]), stored, [45] * b, True)
    assert (np.abs(wide(got) - want) <= attend_tolerance(wide(q), stored, want, dtype)).all()
    # a step of one length, the pair of calls and the fused one: the same bits
    params.sequence_len_offset = 45
    view = mha._update_kv_cache(kv[:, 45:46], params, 0)
    got = attn(q[:, 45:46], view, causal=False)
    want = oracle.attend(wide(q[:, 45:46]), stored, [46] * b)
    assert (np.abs(wide(got) - want) <= attend_tolerance(wide(q), stored, want, dtype)).all()
    assert torch.equal(mha.update_and_attend(q[:, 45:46], kv[:, 45:46], params, 0), got)
    # a ragged step
    lengths = [7, 30, 46, 19, 2]
    params.lengths_per_sample = torch.tensor(lengths, dtype=torch.int32, device=device)
    params.sequence_len_offset = 46
    new = randn((b, 1, 2, h, d), 3, dtype, device, 2.0)
    for i in range(b):
        stored[i, lengths[1 + i]] = oracle.rounded(wide(new[i, 0]))
    view = mha._update_kv_cache(new, params, 0)
    got = attn(q[:, 46:47], view, causal=False)
    want = oracle.attend(wide(q[:, 46:47]), stored, [n + 1 for n in lengths[1:4]])
    assert (np.abs(wide(got) - want) <= attend_tolerance(wide(q), stored, want, dtype)).all()
    assert torch.equal(mha.update_and_attend(q[:, 46:47], new, params, 0), got)
    mha.check_kv_status(device)
    # a position behind the cache is not written, and reported
    params.lengths_per_sample[2] = 60
    before = cache.clone()
    mha.update_and_attend(q[:, 46:47], new, params, 0)
    with pytest.raises(ValueError):
        mha.check_kv_status(device)
    assert torch.equal(cache[2], before[2])


def test_the_ft_caches_stay_as_they_are(device):
    params = InferenceParams(8, fused_ft_kernel=True, kv_bits=4)
    with pytest.raises(ValueError, match="FT caches"):
        mha._update_kv_cache(torch.zeros(1, 2, 2, 2, 32, device=device), params, 0)


# ------------------------------------------------------------- the engine ---


def host():
    return llama.LlamaHost.load(MODEL, "cuda", torch.float32)


def test_a_four_bit_cache_decodes_as_its_rounded_values(device, monkeypatch):
    """Steps over the 4-bit cache against steps over a 16-bit-path cache whose
    rows were rounded when they were written."""
    model = host()
    four, plain = InferenceParams(40, kv_bits=4), InferenceParams(40)
    update = mha._update_kv_cache

    def rounding(kv, params, layer):
        if params.kv_bits == 4:
            return update(kv, params, layer)
        view = update(fp4.dequantize(fp4.quantize(kv.contiguous()), kv.dtype), params, layer)
        return kv if params.sequence_len_offset == 0 else view

    monkeypatch.setattr(llama, "_update_kv_cache", rounding)
    exact = InferenceParams(40)
    ids = torch.tensor([PROMPT], device=device)
    a, b = model.forward(ids, four), model.forward(ids, plain)
    assert torch.equal(a, b)
    monkeypatch.setattr(llama, "_update_kv_cache", update)
    model.forward(ids, exact)
    monkeypatch.setattr(llama, "_update_kv_cache", rounding)
    for step in range(12):
        for p in (four, plain, exact):
            p.sequence_len_offset = len(PROMPT) + step
        token = torch.tensor([[(31 * step + 7) % 128]], device=device)
        a, b = model.forward(token, four, fused_append=step % 2 == 1), model.forward(token, plain)
        assert close(a, b), step
        monkeypatch.setattr(llama, "_update_kv_cache", update)
        assert not close(a, model.forward(token, exact)), "the rounding must show"
        monkeypatch.setattr(llama, "_update_kv_cache", rounding)


def test_four_bit_matrices_compute_as_their_rounded_values(device):
    from safetensors.torch import load_file
    state = {}
    for shard in sorted(MODEL.glob("*.safetensors")):
        state.update(load_file(str(shard)))
    rounded = {k: torch.from_numpy(oracle.rounded(v.double().numpy())).float()
               if k.endswith("_proj.weight") else v for k, v in state.items()}
    shape = llama.LlamaShape.from_config(llama.read_config(MODEL))
    four = llama.LlamaHost(shape, dict(state), "cuda", torch.float32, weight_bits=4)
    plain = llama.LlamaHost(shape, rounded, "cuda", torch.float32)
    assert isinstance(four.layers[0]["wqkv"], fp4.Fp4Tensor)
    for count in (1, 2, 9):  # the few-token products, and the others
        ids = torch.tensor([PROMPT[:count]], device=device)
        a = four.forward(ids, InferenceParams(16), last_token_only=False)
        assert a.shape == (1, count, 128) and close(a, plain.forward(ids, InferenceParams(16), last_token_only=False))
    assert not close(a, host().forward(ids, InferenceParams(16), last_token_only=False)), "the rounding must show"


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
def test_engine_in_four_bits(device, dtype):
    """Prefill, handoff in four bits, decode with scores: the colocated run,
    the fused append and the unfused agree, and the scores are the logits'."""
    count = 9
    engine = Engine(MODEL, "native", "cuda", dtype, kv_bits=4, weight_bits=4)
    tokens, sent, _ = run_split(engine, PROMPT, count)
    assert sent == 8 + 2 * len(PROMPT) * fp4.row_bytes(2, 32)
    first, cache, logits = engine.prefill(PROMPT, count)
    plain = Engine(MODEL, "native", "cuda", dtype, weight_bits=4).prefill(PROMPT, count)
    assert torch.equal(logits, plain[2])  # the prompt attends its own rows
    for layer, kv in plain[1].items():
        assert np.array_equal(wide(fp4.load_kv(cache[layer], len(PROMPT), 2, 32, torch.float32)),
                              oracle.rounded(wide(kv)))
    with pytest.raises(ValueError, match="shape/dtype"):
        engine.decode(first, plain[1], len(PROMPT), count)
    steps, scores = [], []
    assert engine.decode(first, cache, len(PROMPT), count, on_logits=steps.append, on_logprobs=scores.append,
                         top_logprobs=3) == tokens
    engine.fused_append = True
    assert engine.decode(first, cache, len(PROMPT), count) == tokens
    assert len(scores) == count - 1
    for token, logits, got in zip(tokens[1:], steps, scores):
        want = torch.log_softmax(logits.double(), -1)
        # the largest log-probability: sums of 128 terms in fp32, a logarithm and a difference of up to 2^6
        assert abs(float(got.logprob) - float(want[0, token])) <= 128 * 2.0 ** -24 + 2.0 ** -17
        assert torch.equal(got.top_ids, logits.sort(dim=-1, descending=True, stable=True).indices[:, :3])
        assert logits[0, token] == logits.max()
        assert torch.equal(got.top_logprobs[:, 0], got.logprob)


def test_score_matches_the_steps(device):
    """Scoring a whole sequence at once gives what decoding it step by step
    said of the same tokens."""
    count = 8
    engine = Engine(MODEL, "native", "cuda", "float32")
    first, cache, logits = engine.prefill(PROMPT, count)
    steps = [token_logprobs(logits, first, 2)]
    tokens = engine.decode(first, cache, len(PROMPT), count, on_logprobs=steps.append, top_logprobs=2)
    got = engine.score(PROMPT + tokens, top_logprobs=2)
    assert got.logprob.shape == (len(PROMPT) + count - 1,) and got.top_ids.shape == (len(PROMPT) + count - 1, 2)
    scale = LOGITS * 2 * float(logits.abs().max())  # of two logits
    for i, step in enumerate(steps):
        at = len(PROMPT) - 1 + i
        assert torch.equal(got.top_ids[at, :1], step.top_ids[0, :1])
        for a, b in zip(got, step):
            assert a.dtype == torch.int64 or float((a[at] - b[0]).abs().max()) <= scale * 8  # entropy: times -log p < 8
    assert engine.score([4]).logprob.shape == (0,)
    with pytest.raises(ValueError):
        engine.score([])


@pytest.mark.parametrize("weight_bits", [16, 4])
def test_scores_over_a_four_bit_cache_are_the_steps(device, weight_bits):
    """Scoring with ``kv_bits`` 4 gives what steps over the 4-bit cache say of
    the same tokens, and not what the 16-bit cache does."""
    ids = [(37 * i * i + 11 * i + 5) % 128 for i in range(40)]
    engine = Engine(MODEL, "native", "cuda", "float32", kv_bits=4, weight_bits=weight_bits)
    got = engine.score(ids, top_logprobs=2)
    plain = Engine(MODEL, "native", "cuda", "float32", weight_bits=weight_bits).score(ids, top_logprobs=2)
    state, steps, largest = InferenceParams(40, kv_bits=4, attend_stored=True), [], 0.0
    for t in range(39):
        state.sequence_len_offset = t
        logits = engine.model.forward(torch.tensor([[ids[t]]], device=device), state, fused_append=t % 3 == 2)
        steps.append(token_logprobs(logits, torch.tensor([ids[t + 1]], device=device), 2))
        largest = max(largest, float(logits.abs().max()))
    scale = LOGITS * 2 * largest  # of two logits
    for at, step in enumerate(steps):
        for a, b in zip(got, step):
            assert a.dtype == torch.int64 or float((a[at] - b[0]).abs().max()) <= scale * 8  # entropy: times -log p < 8
    assert float((got.logprob - plain.logprob).abs().max()) > scale, "the rounding must show"


def test_engine_refuses_heads_without_whole_blocks(device):
    with pytest.raises(ValueError, match="head_dim"):
        Engine(GOLDEN / "tiny_llama", "native", "cuda", "float16", kv_bits=4)  # head_dim 16


@pytest.mark.timeout(600)
def test_pilot_in_four_bits(tmp_path):
    result = launch(tmp_path / "out", "--kv-bits", "4", "--weight-bits", "4", "--logprobs", "--fused-append")
    assert result.returncode == 0, result.stderr[-4000:]
    records = [json.loads(s) for s in (tmp_path / "out" / "requests.jsonl").read_text().splitlines()]
    assert [r["output_tokens"] for r in records] == [1, 1, 4, 3]
    for r in records:
        assert r["colocated_matches"]
        assert r["kv_packet_bytes"] == 8 + 2 * r["input_tokens"] * fp4.row_bytes(2, 32)
        assert len(r["decode"]["logprobs"]) == len(r["decode"]["entropies"]) == r["output_tokens"] - 1
        # a greedy token has at least the mean probability, and -log p of the likeliest is at most the entropy
        assert all(-np.log(128) - 1e-4 <= p <= 0 and -p <= e + 1e-4
                   for p, e in zip(r["decode"]["logprobs"], r["decode"]["entropies"]))
