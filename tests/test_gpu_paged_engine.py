"""The engine, the model host and the attention module over paged caches: the
tokens and logits of the plain caches, prompts in chunks, several requests in
one pool, and handoffs between paged and plain sides."""
import json

import pytest
import torch

from hexgen2_amd import mha, ops, paged
from hexgen2_amd.engine import Engine
from hexgen2_amd.generation import InferenceParams
from hexgen2_amd.llama import LlamaHost, LlamaShape
from tests.test_gpu_engine import GOLDEN, GREEDY, check_logits, run_split
from tests.test_gpu_pilot import check_records, launch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("chunk", [0, 1, 3])
def test_fixture_tokens_over_pages(device, dtype, chunk):
    engine = Engine(GOLDEN / "fixture_seed17", "native", "cuda", dtype, page_size=16, prefill_chunk=chunk)
    for case in GREEDY["fixture_seed17"]:
        tokens, sent, logits = run_split(engine, case["prompt"], case["max_new_tokens"])
        assert tokens == case["hf_fp32_tokens"]
        elem = 4 if dtype == "float32" else 2
        assert sent == 8 + 2 * len(case["prompt"]) * 2 * 2 * 32 * elem  # the packet is that of the plain caches
        check_logits("fixture_seed17", case["prompt"], dtype, logits)


@pytest.mark.parametrize("dtype", ["float16", "float32"])
def test_tiny_llama_over_pages(device, dtype):
    case = GREEDY["tiny_llama"][0]
    engine = Engine(GOLDEN / "tiny_llama", "native", "cuda", dtype, page_size=16, prefill_chunk=5)
    tokens, _, logits = run_split(engine, case["prompt"], case["max_new_tokens"])
    assert tokens == case["hf_fp32_tokens"]
    check_logits("tiny_llama", case["prompt"], dtype, logits)


def test_paged_and_plain_sides_hand_over_to_each_other(device):
    case = GREEDY["tiny_llama"][0]
    sides = [Engine(GOLDEN / "tiny_llama", "native", "cuda", "float32", page_size=n) for n in (0, 32)]
    for prefill, decode in (sides, sides[::-1]):
        first, cache, _ = prefill.prefill(case["prompt"], case["max_new_tokens"])
        assert decode.decode(first, cache, len(case["prompt"]), case["max_new_tokens"]) == case["hf_fp32_tokens"]
    scores = [e.score(case["prompt"], 3) for e in sides]
    for a, b in zip(*scores):
        assert torch.allclose(a.float(), b.float(), atol=1e-4)


def random_host(dtype, scaling=None, heads=8, kv_heads=2, d=64, layers=2, seed=0):
    g = torch.Generator().manual_seed(seed)
    hidden, mid, vocab = heads * d, 192, 211

    def w(*shape):
        return torch.randn(shape, generator=g) * shape[-1] ** -0.5

    weights = {"model.embed_tokens.weight": w(vocab, hidden) * hidden ** 0.5, "model.norm.weight": torch.ones(hidden),
               "lm_head.weight": w(vocab, hidden)}
    for i in range(layers):
        p = f"model.layers.{i}."
        weights.update({p + "input_layernorm.weight": torch.ones(hidden), p + "post_attention_layernorm.weight": torch.ones(hidden),
                        p + "self_attn.q_proj.weight": w(hidden, hidden), p + "self_attn.k_proj.weight": w(kv_heads * d, hidden),
                        p + "self_attn.v_proj.weight": w(kv_heads * d, hidden), p + "self_attn.o_proj.weight": w(hidden, hidden),
                        p + "mlp.gate_proj.weight": w(mid, hidden), p + "mlp.up_proj.weight": w(mid, hidden),
                        p + "mlp.down_proj.weight": w(hidden, mid)})
    shape = LlamaShape(vocab, hidden, mid, layers, heads, kv_heads, rope_scaling=scaling, max_position_embeddings=64)
    return LlamaHost(shape, weights, "cuda", dtype)


SCALINGS = [None, {"rope_type": "linear", "factor": 4.0},
            {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
             "original_max_position_embeddings": 64},
            {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32}]


@pytest.mark.parametrize("scaling", SCALINGS)
def test_logits_of_paged_and_plain_caches_agree(device, scaling):
    """Prompt, a second chunk and decode steps in float32, each against one
    forward pass of the plain caches over all tokens."""
    host = random_host(torch.float32, scaling)
    ids = torch.randint(0, 211, (2, 90), generator=torch.Generator().manual_seed(3)).cuda()
    plain = InferenceParams(max_sequence_len=128, max_batch_size=2)
    want = host.forward(ids, plain, last_token_only=False)
    pages = InferenceParams(max_sequence_len=128, max_batch_size=2, page_size=16)
    got = []
    for at, n in ((0, 50), (50, 37), (87, 1), (88, 1), (89, 1)):
        pages.sequence_len_offset = at
        got.append(host.forward(ids[:, at:at + n], pages, last_token_only=False))
    assert torch.allclose(torch.cat(got, dim=1), want, atol=2e-4)
    assert pages.page_tables.shape == (2, 8) and len(pages.key_value_memory_dict) == 2


def test_ragged_decode_over_pages(device):
    """lengths_per_sample, as the plain caches take it."""
    host = random_host(torch.float32)
    ids = torch.randint(0, 211, (3, 40), generator=torch.Generator().manual_seed(4)).cuda()
    lens = [40, 17, 3]
    step = torch.randint(0, 211, (3, 1), generator=torch.Generator().manual_seed(5)).cuda()
    outs = []
    for page in (0, 32):
        params = InferenceParams(max_sequence_len=64, max_batch_size=3, page_size=page)
        host.forward(ids, params)
        params.sequence_len_offset = 40
        params.lengths_per_sample = torch.tensor(lens, dtype=torch.int32, device="cuda")
        outs.append(host.forward(step, params))
    assert torch.allclose(outs[0], outs[1], atol=2e-4)
    assert ops.device_status(device) & ops._lib.STATUS_ERRORS == 0


def test_the_attention_module_over_pages(device):
    """_update_kv_cache, FlashCrossAttention and update_and_attend, call by call."""
    g = torch.Generator().manual_seed(6)
    attn = mha.FlashCrossAttention(causal=True, softmax_scale=0.1)
    sides = [InferenceParams(max_sequence_len=100, max_batch_size=4, batch_size_offset=1, page_size=n) for n in (0, 16)]
    for offset, n, causal in ((0, 37, None), (37, 1, False), (38, 1, False)):
        q = torch.randn(3, n, 8, 64, generator=g).half().cuda()
        kv = torch.randn(3, n, 2, 2, 64, generator=g).half().cuda()
        out = []
        for params in sides:
            params.sequence_len_offset = offset
            if offset == 38:
                out.append(mha.update_and_attend(q, kv, params, 0, 0.1))
            else:
                out.append(attn(q, mha._update_kv_cache(kv, params, 0), causal=causal))
        assert (out[0].float() - out[1].float()).abs().max() < 4e-3
    rows = paged.pack_live([sides[1].key_value_memory_dict[0]], sides[1].page_tables[1:], [39] * 3)
    assert torch.equal(rows[0].view(3, 39, 2, 2, 64), sides[0].key_value_memory_dict[0][1:4, :39])


@pytest.mark.parametrize("dtype,options", [("float32", {}), ("float32", dict(step_tokens=7, chunk=3)), ("float16", dict(chunk=4)),
                                           ("float32", dict(pool_pages=2, step_tokens=5))])
def test_generate_answers_as_one_request_at_a_time(device, dtype, options):
    options = dict(options)
    engine = Engine(GOLDEN / "fixture_seed17", "native", "cuda", dtype, page_size=16, prefill_chunk=options.pop("chunk", 0))
    cases = GREEDY["fixture_seed17"] * 3
    told = []
    answers = engine.generate([c["prompt"] for c in cases], [c["max_new_tokens"] for c in cases],
                              on_token=lambda i, t: told.append((i, t)), **options)
    assert answers == [c["hf_fp32_tokens"] for c in cases]
    assert sorted(told, key=lambda x: x[0]) == [(i, t) for i, a in enumerate(answers) for t in a]
    assert engine.generate([], 3) == []


def test_generate_refuses_what_cannot_run(device):
    engine = Engine(GOLDEN / "tiny_llama", "native", "cuda", "float16", page_size=16)
    with pytest.raises(ValueError, match="pool of 1 pages"):
        engine.generate([[1] * 20], 4, pool_pages=1)
    with pytest.raises(ValueError, match="needs a token"):
        engine.generate([[1], []], 4)
    with pytest.raises(ValueError, match="needs a token"):
        engine.generate([[1], [2]], [4, 0])
    with pytest.raises(ValueError, match="step of 0"):
        engine.generate([[1]], 4, step_tokens=0)
    with pytest.raises(ValueError, match="needs a token"):
        engine.prefill([], 4)
    pool = engine._pool(1)
    with pytest.raises(ValueError, match="pools of 1 layers"):
        engine.model.forward_pages(torch.tensor([[1]], device=device), pool[:1], torch.zeros((1, 1), dtype=torch.int32, device=device),
                                   torch.zeros(1, dtype=torch.int32, device=device), max_seqlen=1)
    with pytest.raises(ValueError, match="page_size"):
        Engine(GOLDEN / "tiny_llama", "native", "cuda", "float16").generate([[1]], 4)


@pytest.mark.timeout(600)
def test_pilot_over_pages(tmp_path):
    result = launch(tmp_path / "out", "--page-size", "16", "--prefill-chunk", "3")
    assert result.returncode == 0, result.stderr[-4000:]
    check_records(tmp_path / "out", 2, golden=True)
