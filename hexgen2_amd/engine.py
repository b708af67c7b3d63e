"""Prefill/decode engine with the KV handoff on the GPU.

Mirrors the pilot's ``Engine`` (hexgen2/model.py:22-124): same constructor,
``prefill(input_ids, max_new_tokens) -> (first_token, cache, logits)`` and
``decode(first_token, cache, prompt_length, max_new_tokens, on_token=None)``,
same cache dict contract ``{layer: [1, L, 2, kv_heads, head_dim]}`` and the
same validation errors.  What changes is where the bytes go:

* prefill ends with ONE hexkv pack launch that gathers the live rows of every
  layer into one contiguous handoff buffer; the returned dict holds
  per-layer views of that buffer (model.py:81 did one copy per layer);
* decode starts with ONE hexkv unpack launch that scatters the received
  layers into a single preallocated decode cache (model.py:104-108 allocated
  and copied per layer);
* each decode step appends and attends through hexkv (mha.py:286, 568-569).

Additions: ``kv_bits`` 4 keeps and hands over the caches in four bits (uint8 rows,
``{layer: [1, L, row_bytes]}``; a prompt attends its own keys unrounded),
``weight_bits`` 4 the layers' matrices, and ``decode(on_logprobs=...)`` and
``score`` report what the logits say of the tokens.  ``page_size`` keeps the caches in
pages (the handed-off dict is the same, so either side may), ``prefill_chunk`` lets a
prompt go through in chunks of that many tokens, and ``generate`` answers several prompts at
once over one pool.
"""
from __future__ import annotations

import hashlib
import json
from collections import deque
from pathlib import Path

import torch

from . import fp4, ops, paged
from .generation import CacheState
from .llama import LlamaHost, LlamaShape, read_config
from .logprobs import TokenLogprobs, token_logprobs
from .mha import check_kv_status


# Packed handoff buffers at or above this size are allocated per layer, so
# that each stays an allocation another process can map (below 2 GiB).
PER_LAYER_HANDOFF_BYTES = 1 << 30


def model_identity(model_dir) -> dict:
    """SHA-256 of every checkpoint/config file and of their listing, as the
    pilot records it (hexgen2/record.py:36-45)."""
    files = sorted(p for p in Path(model_dir).iterdir() if p.is_file() and (
        p.suffix in {".safetensors", ".json"} or p.name == "tokenizer.model"))
    hashes = {p.name: hashlib.sha256(p.read_bytes()).hexdigest() for p in files}
    if not any(name.endswith(".safetensors") for name in hashes):
        raise ValueError("No safetensors checkpoint in model directory")
    return {"files": hashes, "sha256": hashlib.sha256(json.dumps(hashes, sort_keys=True).encode()).hexdigest()}


class Engine:
    def __init__(self, model_dir, engine="native", device="cuda", dtype="float16",
                 fused_append: bool = False, *, kv_bits: int = 16, weight_bits: int = 16, page_size: int = 0,
                 prefill_chunk: int = 0):
        if kv_bits not in (16, 4) or weight_bits not in (16, 4):
            raise ValueError(f"caches and weights hold 16 bits (their dtype) or 4, got {kv_bits} and {weight_bits}")
        if page_size and (page_size < 16 or page_size & (page_size - 1) or kv_bits != 16):
            raise ValueError(f"pages hold a power of two of positions from 16 on, in the data type (got {page_size} "
                             f"positions of {kv_bits} bits)")
        if prefill_chunk < 0 or (prefill_chunk and not page_size):
            raise ValueError(f"prompts go in chunks of {prefill_chunk} tokens over paged caches only (page_size)")
        self.device, self.dtype = torch.device(device), getattr(torch, dtype)
        self.shape = LlamaShape.from_config(read_config(model_dir))
        self.identity = model_identity(model_dir)
        self.kind = engine
        if engine != "native":
            raise ValueError("Only the native engine runs on the hexkv data path; the "
                             "hf-reference engine is the reference's CPU validator")
        if self.device.type != "cuda" or not torch.cuda.is_available():
            raise ValueError("The hexkv engine requires a HIP GPU (torch.cuda on ROCm)")
        self.kv_bits, self.page_size, self.prefill_chunk = kv_bits, page_size, prefill_chunk
        self._cache_row()  # (refuses heads that a 4-bit cache cannot hold)
        self.model = LlamaHost.load(model_dir, self.device, self.dtype, weight_bits)
        self.fused_append = fused_append
        self.config = self.shape

    def _cache_geometry(self):
        s = self.shape
        return s.num_hidden_layers, s.num_key_value_heads, s.head_dim

    def _cache_row(self):
        """Shape and type of one position's cache row."""
        _, kv_heads, head_dim = self._cache_geometry()
        if self.kv_bits == 4:
            return (fp4.row_bytes(kv_heads, head_dim),), torch.uint8
        return (2, kv_heads, head_dim), self.dtype

    @torch.inference_mode()
    def prefill(self, input_ids, max_new_tokens):
        if self.page_size and not len(input_ids):
            raise ValueError("prefill needs a token")
        ids = torch.tensor([input_ids], dtype=torch.long, device=self.device)
        state = CacheState(len(input_ids) + max_new_tokens, kv_bits=self.kv_bits, page_size=self.page_size)
        chunk = self.prefill_chunk or len(input_ids)
        for state.sequence_len_offset in range(0, len(input_ids), chunk) if self.page_size else (0,):
            at = state.sequence_len_offset
            logits = self.model.forward(ids[:, at:at + chunk], inference_params=state, last_token_only=True)
        n_layers = len(state.key_value_memory_dict)
        layers = [state.key_value_memory_dict[i] for i in range(n_layers)]
        # Send only initialized prompt positions, never the unused capacity:
        # one launch gathers every layer into one handoff buffer (per-layer
        # buffers when it would be too large to map from another process).
        row_shape = layers[0].shape[2:]
        nbytes = n_layers * len(input_ids) * layers[0][0, 0].numel() * layers[0].element_size()
        out = None
        if nbytes >= PER_LAYER_HANDOFF_BYTES:
            out = [torch.empty((len(input_ids), *row_shape), dtype=layers[0].dtype, device=self.device)
                   for _ in range(n_layers)]
        if self.page_size:
            packed = paged.pack_live(layers, state.page_tables, [len(input_ids)], out=out)
        else:
            packed = ops.pack_live(layers, [len(input_ids)], out=out)
        cache = {i: packed[i].unsqueeze(0) for i in range(n_layers)}
        return logits.argmax(-1), cache, logits

    @torch.inference_mode()
    def decode(self, first_token, cache, prompt_length, max_new_tokens, on_token=None, *, on_logits=None,
               on_logprobs=None, top_logprobs=0):
        """Greedy decode from the handed-off cache (model.py:86-120).
        ``on_logits`` (an addition) receives each decode step's logits
        ``[1, vocab]``, for logit-level checks; ``on_logprobs`` (another) each
        decode step's ``TokenLogprobs`` of the token taken, with the
        ``top_logprobs`` likeliest ones.  (The first token's are
        ``token_logprobs`` of the logits ``prefill`` returns.)"""
        token = first_token.to(self.device).reshape(1)
        generated = [int(token.item())]
        if on_token:
            on_token(generated[-1])
        n_layers = self._cache_geometry()[0]
        row_shape, row_dtype = self._cache_row()
        if set(cache) != set(range(n_layers)):
            raise ValueError("KV cache does not match the configured layer count")
        expected = (1, prompt_length, *row_shape)
        for value in cache.values():
            if tuple(value.shape) != expected or value.dtype != row_dtype:
                raise ValueError("KV cache shape/dtype does not match checkpoint and prompt")
        state = CacheState(prompt_length + max_new_tokens, kv_bits=self.kv_bits, page_size=self.page_size)
        state.sequence_len_offset = prompt_length
        live = [cache[i].to(self.device) for i in range(n_layers)]
        live = [t if t.is_contiguous() else t.contiguous() for t in live]
        # One decode cache for all layers; rows >= prompt_length stay
        # uninitialised as in model.py:105.
        if self.page_size:
            full = self._pool(paged.pages_for(state.max_sequence_len, self.page_size))
            state.page_tables = torch.arange(full.shape[1], dtype=torch.int32, device=self.device)[None]
            paged.unpack_live(live, full, state.page_tables, [prompt_length])
        else:
            full = torch.empty((n_layers, 1, state.max_sequence_len, *row_shape), device=self.device, dtype=row_dtype)
            ops.unpack_live(live, full, [prompt_length])
        for i in range(n_layers):
            state.key_value_memory_dict[i] = full[i]
        ops.device_status(self.device)  # report only what this decode's kernels meet
        for _ in range(max_new_tokens - 1):
            logits = self.model.forward(token[:, None], inference_params=state, last_token_only=True,
                                        fused_append=self.fused_append)
            state.sequence_len_offset += 1
            if on_logits:
                on_logits(logits)
            token = logits.argmax(-1)
            if on_logprobs:
                on_logprobs(token_logprobs(logits, token, top_logprobs))
            generated.append(int(token.item()))
            # the token read synchronised: report any out-of-contract device
            # position the step's kernels met (mha.py:281-282's assert)
            check_kv_status(self.device)
            if on_token:
                on_token(generated[-1])
        return generated

    def _pool(self, n_pages: int) -> torch.Tensor:
        """A pool of pages for every layer, stacked."""
        n_layers, kv_heads, head_dim = self._cache_geometry()
        return paged.kv_pages(n_pages, self.page_size, kv_heads, head_dim, self.dtype, self.device, layers=n_layers)

    @torch.inference_mode()
    def generate(self, prompts, max_new_tokens, *, pool_pages=None, step_tokens=512, on_token=None):
        """Greedy answers of up to ``max_new_tokens`` (one number, or one a prompt) to
        several prompts at once, over one pool of ``pool_pages`` pages (default: enough for
        all of them).  Every step is one forward pass: the next token of each sequence that
        is past its prompt, and of the others' prompts as many tokens as make up
        ``step_tokens`` (``prefill_chunk`` at most a sequence).  A prompt waits until the pool
        has the pages that it and its answer need; they are given back when it is
        answered.  ``on_token(prompt, token)`` is told of each token.  Returns the
        answers in the prompts' order."""
        if not self.page_size:
            raise ValueError("generate works over paged caches (Engine(page_size=...))")
        prompts = [list(p) for p in prompts]
        limits = [int(max_new_tokens)] * len(prompts) if isinstance(max_new_tokens, int) else [int(n) for n in max_new_tokens]
        if len(limits) != len(prompts) or any(not p for p in prompts) or any(n < 1 for n in limits):
            raise ValueError("every prompt needs a token, and an answer of at least one")
        if step_tokens < 1:
            raise ValueError(f"a step of {step_tokens} tokens")
        need = [paged.pages_for(len(p) + n - 1, self.page_size) for p, n in zip(prompts, limits)]
        total = sum(need) if pool_pages is None else int(pool_pages)
        if need and total < max(need):
            raise ValueError(f"a pool of {total} pages for a prompt that needs {max(need)}")
        if not prompts:
            return []
        pool = self._pool(total)
        free, waiting, running = list(range(total)), deque(range(len(prompts))), []  # running: [prompt, rows cached, pages]
        answers = [[] for _ in prompts]
        ops.device_status(self.device)  # report only what these steps' kernels meet
        while waiting or running:
            while waiting and need[waiting[0]] <= len(free):
                i = waiting.popleft()
                running.append([i, 0, [free.pop() for _ in range(need[i])]])
            budget = step_tokens - sum(done >= len(prompts[i]) for i, done, _ in running)
            step = []  # (entry, its tokens)
            for entry in running:
                i, done, _ = entry
                if done >= len(prompts[i]):
                    step.append((entry, answers[i][-1:]))
                    continue
                count = min(len(prompts[i]) - done, budget, self.prefill_chunk or step_tokens)
                if count > 0 or not step:
                    count = max(count, 1)
                    step.append((entry, prompts[i][done:done + count]))
                    budget -= count
            width = max(len(entry[2]) for entry, _ in step)
            bounds = [0]
            for _, tokens in step:
                bounds.append(bounds[-1] + len(tokens))
            starts = [entry[1] for entry, _ in step]
            tables = [entry[2] + [-1] * (width - len(entry[2])) for entry, _ in step]
            longest = max(start + len(tokens) for start, (_, tokens) in zip(starts, step))
            most = max(len(tokens) for _, tokens in step)

            def int32(values):
                return torch.tensor(values, dtype=torch.int32, device=self.device)

            ids = torch.tensor([[t for _, tokens in step for t in tokens]], dtype=torch.long, device=self.device)
            last = torch.tensor(bounds[1:], dtype=torch.long, device=self.device) - 1
            logits = self.model.forward_pages(ids, pool, int32(tables), int32(starts), max_seqlen=longest,
                                              cu_tokens=int32(bounds) if most > 1 else None, max_tokens=most, rows=last)
            picked = logits.argmax(-1).tolist()
            check_kv_status(self.device)
            for (entry, tokens), token in zip(step, picked):
                i = entry[0]
                entry[1] += len(tokens)
                if entry[1] < len(prompts[i]):
                    continue
                answers[i].append(token)
                if on_token:
                    on_token(i, token)
                if len(answers[i]) == limits[i]:
                    free.extend(entry[2])
                    running.remove(entry)
        return answers

    @torch.inference_mode()
    def score(self, input_ids, top_logprobs=0) -> TokenLogprobs:
        """What the model says of a sequence's tokens: entry t of each result
        belongs to ``input_ids[t + 1]`` after the t + 1 tokens before it.  With
        ``kv_bits`` 4 every token attends its rows as the cache holds them, as
        a decode step does (``prefill`` attends them unrounded)."""
        if not len(input_ids):
            raise ValueError("score needs a token")
        ids = torch.tensor([input_ids], dtype=torch.long, device=self.device)
        state = CacheState(len(input_ids), kv_bits=self.kv_bits, attend_stored=True, page_size=self.page_size)
        logits = self.model.forward(ids, inference_params=state, last_token_only=False)
        return token_logprobs(logits[0, :-1], ids[0, 1:], top_logprobs)

    def synchronize(self):
        if self.device.type == "cuda":
            torch.cuda.synchronize(self.device)
