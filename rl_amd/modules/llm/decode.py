"""Graph-captured GPT-2 decode for RLHF rollouts on MI355X.

The HF single-token decode path can't be hipGraph-captured on this
stack (``StaticCache`` + ROCm 7.2 segfaults, and ``generate`` burns
milliseconds of host logic per token), so :class:`GraphedGPT2Decoder`
reimplements the GPT-2 decode step directly on the model's own
parameters with manually-managed static KV buffers: one prefill
(ordinary HF forward) and then ONE captured graph replay per generated
token — embedding lookup, 12 blocks of LN/attention-over-static-KV/MLP,
final LN, tied-lm-head logits, multinomial sampling and all buffer
bookkeeping.

The captured kernels read the policy's bf16 weight CACHES (refreshed
once per training iteration via :meth:`refresh_weights`), so the same
graph keeps decoding as training updates the fp32 masters.

Reference analog: torchrl's vLLM-backed generation
(torchrl/modules/llm/backends/vllm*); here the engine is a hand-rolled
static-KV loop because the image has no vLLM and HF's static path dies.
Numerics validated against the eager HF forward in
tests/test_llm_bench.py (same sampling distribution as
``generate(do_sample=True, top_k=0)``).
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn.functional as F

from ... import ops
from ...tensordict import TensorDict
from .paged_cache import PagedKVCache

__all__ = ["GraphedGPT2Decoder", "PagedGPT2Decoder"]


class GraphedGPT2Decoder:
    def __init__(self, model, batch: int, max_len: int, device,
                 dtype=torch.bfloat16):
        self._bind(model, batch, max_len, device, dtype)
        # static KV + bookkeeping buffers
        kv = (self.L, self.B, self.nh, self.T, self.dh)
        self.K = torch.zeros(kv, device=device, dtype=dtype)
        self.Vv = torch.zeros(kv, device=device, dtype=dtype)
        self.mask = torch.full((self.T,), float("-inf"), device=device)
        self.cur = torch.zeros(self.B, 1, dtype=torch.long, device=device)
        self.pos = torch.zeros(1, dtype=torch.long, device=device)
        self.pos_out = torch.zeros(1, dtype=torch.long, device=device)
        self.gen_buf = torch.zeros(self.B, self.T, dtype=torch.long,
                                   device=device)
        self._graph = None

    def _bind(self, model, batch, max_len, device, dtype) -> None:
        self.model = model
        self.cfg = model.config
        self.B = batch
        self.T = max_len
        self.device = device
        self.dtype = dtype
        c = self.cfg
        self.L, self.nh, self.E = c.n_layer, c.n_head, c.n_embd
        self.dh = self.E // self.nh
        self.V = c.vocab_size
        tr = model.transformer
        self._blocks = list(tr.h)
        self._tr = tr
        # bf16 weight caches (refreshed per training iteration)
        self._w = {}
        self.refresh_weights()

    # ------------------------------------------------------------------ #
    def refresh_weights(self) -> None:
        """Re-cast the decode weight caches from the live parameters
        (call once per training iteration, after the optimizer step)."""
        bf = self.dtype
        w = self._w
        tr = self._tr
        first = not w
        def put(name, t, dtype):
            t = t.detach().to(dtype)
            if first:
                w[name] = t.clone()
            else:
                w[name].copy_(t)
        put("wte", tr.wte.weight, bf)
        put("wpe", tr.wpe.weight, bf)
        put("lnf_w", tr.ln_f.weight, torch.float32)
        put("lnf_b", tr.ln_f.bias, torch.float32)
        for i, blk in enumerate(self._blocks):
            put(f"ln1_w{i}", blk.ln_1.weight, torch.float32)
            put(f"ln1_b{i}", blk.ln_1.bias, torch.float32)
            put(f"attn_w{i}", blk.attn.c_attn.weight, bf)   # [E, 3E]
            put(f"attn_b{i}", blk.attn.c_attn.bias, bf)
            put(f"proj_w{i}", blk.attn.c_proj.weight, bf)   # [E, E]
            put(f"proj_b{i}", blk.attn.c_proj.bias, bf)
            put(f"ln2_w{i}", blk.ln_2.weight, torch.float32)
            put(f"ln2_b{i}", blk.ln_2.bias, torch.float32)
            put(f"fc_w{i}", blk.mlp.c_fc.weight, bf)        # [E, 4E]
            put(f"fc_b{i}", blk.mlp.c_fc.bias, bf)
            put(f"fc2_w{i}", blk.mlp.c_proj.weight, bf)     # [4E, E]
            put(f"fc2_b{i}", blk.mlp.c_proj.bias, bf)

    # ------------------------------------------------------------------ #
    def _step_logits(self) -> torch.Tensor:
        """One decode forward over the static KV: [B, V] fp32 logits
        for the token ids in ``self.cur`` at position ``self.pos``."""
        w = self._w
        B, nh, dh, E = self.B, self.nh, self.dh, self.E
        eps = self.cfg.layer_norm_epsilon
        # the new token becomes attendable
        self.mask.index_fill_(0, self.pos, 0.0)
        x = (w["wte"].index_select(0, self.cur.reshape(-1))
             + w["wpe"].index_select(0, self.pos)).reshape(B, 1, E)
        scale = 1.0 / float(dh) ** 0.5
        for i in range(self.L):
            xn = F.layer_norm(x.float(), (E,), w[f"ln1_w{i}"],
                              w[f"ln1_b{i}"], eps).to(self.dtype)
            qkv = torch.addmm(w[f"attn_b{i}"], xn.reshape(B, E),
                              w[f"attn_w{i}"])
            q, k, v = qkv.split(E, dim=-1)
            q = q.reshape(B, nh, 1, dh)
            k = k.reshape(B, 1, nh, dh).transpose(1, 2)
            v = v.reshape(B, 1, nh, dh).transpose(1, 2)
            self.K[i].index_copy_(2, self.pos, k)
            self.Vv[i].index_copy_(2, self.pos, v)
            att = torch.matmul(q, self.K[i].transpose(-1, -2)).float()
            att = att * scale + self.mask
            probs = att.softmax(-1).to(self.dtype)
            o = torch.matmul(probs, self.Vv[i])      # [B, nh, 1, dh]
            o = o.transpose(1, 2).reshape(B, E)
            x = x + torch.addmm(w[f"proj_b{i}"], o,
                                w[f"proj_w{i}"]).reshape(B, 1, E)
            xn = F.layer_norm(x.float(), (E,), w[f"ln2_w{i}"],
                              w[f"ln2_b{i}"], eps).to(self.dtype)
            h = torch.addmm(w[f"fc_b{i}"], xn.reshape(B, E), w[f"fc_w{i}"])
            h = F.gelu(h, approximate="tanh")
            x = x + torch.addmm(w[f"fc2_b{i}"], h,
                                w[f"fc2_w{i}"]).reshape(B, 1, E)
        xn = F.layer_norm(x.float(), (E,), w["lnf_w"], w["lnf_b"], eps)
        logits = torch.matmul(xn.to(self.dtype).reshape(B, E),
                              w["wte"].t())
        return logits.float()

    def _decode_body(self) -> None:
        logits = self._step_logits()
        nxt = torch.multinomial(torch.softmax(logits, -1), 1)
        self.cur.copy_(nxt)
        self.gen_buf.index_copy_(1, self.pos_out, nxt)
        self.pos.add_(1)
        self.pos_out.add_(1)

    # ------------------------------------------------------------------ #
    def prefill(self, prompts: torch.Tensor) -> None:
        """HF forward over the prompts; copies its KV into the static
        buffers and samples the first generated token."""
        P = prompts.shape[1]
        with torch.no_grad(), torch.autocast(
            "cuda", dtype=self.dtype, cache_enabled=False,
            enabled=prompts.is_cuda,
        ):
            out = self.model(input_ids=prompts, use_cache=True)
        past = out.past_key_values
        for i in range(self.L):
            if hasattr(past, "layers"):  # transformers >= 4.54 Cache
                k, v = past.layers[i].keys, past.layers[i].values
            elif hasattr(past, "key_cache"):
                k, v = past.key_cache[i], past.value_cache[i]
            else:
                k, v = past[i]
            self.K[i, :, :, :P] = k.to(self.dtype)
            self.Vv[i, :, :, :P] = v.to(self.dtype)
        self.mask.fill_(float("-inf"))
        self.mask[:P] = 0.0
        logits = out.logits[:, -1].float()
        first = torch.multinomial(torch.softmax(logits, -1), 1)
        self.cur.copy_(first)
        self.gen_buf[:, 0:1] = first
        self.pos.fill_(P)
        self.pos_out.fill_(1)

    def capture(self) -> bool:
        """hipGraph-capture the decode step (after at least one
        prefill).  Returns False (eager fallback stays) on failure."""
        try:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side), torch.no_grad():
                for _ in range(3):
                    self._decode_body()
            torch.cuda.current_stream().wait_stream(side)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g), torch.no_grad():
                self._decode_body()
            self._graph = g
            return True
        except Exception:
            self._graph = None
            return False

    def rollout(self, prompts: torch.Tensor, gen_tokens: int) -> torch.Tensor:
        """Generate ``gen_tokens`` tokens; returns [B, P + G] ids."""
        self.prefill(prompts)
        with torch.no_grad():
            for _ in range(gen_tokens - 1):
                if self._graph is not None:
                    self._graph.replay()
                else:
                    self._decode_body()
        return torch.cat(
            [prompts, self.gen_buf[:, :gen_tokens]], dim=1
        )


class PagedGPT2Decoder(GraphedGPT2Decoder):
    """GPT-2 decode over a :class:`PagedKVCache`: prompts of any lengths in
    one batch, an optional end token, and the behavior log-probs that the
    policy losses need, recorded while sampling.

    Per generated token and layer: one cache append
    (:func:`rl_amd.ops.paged_kv_append`) and one attention over each
    sequence's own length (:func:`rl_amd.ops.paged_attention_decode`), where
    :class:`GraphedGPT2Decoder` attends over ``max_len`` for every sequence.
    There is no dropout, whatever mode the model is in.
    After :meth:`capture` each token is one graph replay; a sequence that has
    produced ``eos_token_id`` stops writing to its cache.

    Args:
        model: a transformers GPT-2 with tied LM head, tanh GELU and attention
            scores over ``sqrt(dim)`` (the architecture's defaults).
        batch: sequences per rollout.
        max_len: longest prompt plus response; at most the model's positions.
        temperature: of the sampling and of the recorded log-probs.
        eos_token_id: stop a sequence after this token; None: never.
        page_size: positions per cache page (a power of two).
    """

    def __init__(self, model, batch: int, max_len: int, device, dtype=torch.bfloat16, *,
                 temperature: float = 1.0, eos_token_id: Optional[int] = None, page_size: int = 16):
        if max_len > model.config.n_positions:
            raise ValueError(
                f"PagedGPT2Decoder: max_len {max_len} exceeds the model's {model.config.n_positions} positions")
        c = model.config
        if (
            c.activation_function not in self._TANH_GELU
            or not c.scale_attn_weights
            or c.scale_attn_by_inverse_layer_idx
        ):
            raise ValueError(
                "PagedGPT2Decoder: the decode step is that of a tanh GELU and scores over sqrt(dim), not of "
                f"activation_function={c.activation_function!r}, scale_attn_weights={c.scale_attn_weights}, "
                f"scale_attn_by_inverse_layer_idx={c.scale_attn_by_inverse_layer_idx}")
        if model.lm_head.weight.data_ptr() != model.transformer.wte.weight.data_ptr():
            raise ValueError("PagedGPT2Decoder: the LM head must be tied to the token embedding")
        if eos_token_id is not None and not 0 <= eos_token_id < model.config.vocab_size:
            raise ValueError(
                f"PagedGPT2Decoder: eos_token_id {eos_token_id} is not in the vocabulary of {model.config.vocab_size}")
        if not 1e-30 <= temperature <= 1e30:
            raise ValueError(f"PagedGPT2Decoder: temperature must be positive, got {temperature}")
        self._bind(model, batch, max_len, device, dtype)
        self.temperature = temperature
        self.eos_token_id = eos_token_id
        self.cache = PagedKVCache(
            self.L, batch * -(-max_len // page_size), self.nh, self.dh, batch=batch,
            max_length=max_len, page_size=page_size, dtype=dtype, device=device)
        self.cur = torch.zeros(batch, dtype=torch.long, device=device)
        self.active = torch.ones(batch, dtype=torch.int32, device=device)
        self.pos_out = torch.zeros(1, dtype=torch.long, device=device)
        self.gen_buf = torch.zeros(batch, max_len, dtype=torch.long, device=device)
        self.lp_buf = torch.zeros(batch, max_len, dtype=torch.float32, device=device)
        self.mask_buf = torch.zeros(batch, max_len, dtype=torch.bool, device=device)
        # the sampling scores, padded so that an argmax goes in two short stages
        self._chunks = -(-self.V // self._CHUNK)
        self._scores = torch.full((batch, self._chunks * self._CHUNK), float("-inf"), device=device)
        self._graph = None

    _CHUNK = 512
    _TANH_GELU = ("gelu_new", "gelu_pytorch_tanh", "gelu_fast", "gelu_accurate")

    def _draw(self, logits: torch.Tensor) -> torch.Tensor:
        """A token of ``softmax(logits / temperature)`` per row: the argmax of
        ``logits / temperature - log(e)`` with ``e`` exponential.  (Not
        ``multinomial``: its validity checks reduce the whole tensor over many
        blocks, which puts memory-set nodes into a captured graph, and those
        have given wrong results on later replays; short rows are reduced
        without them.)"""
        noise = torch.empty_like(logits).exponential_().log_()
        torch.sub(logits / self.temperature, noise, out=self._scores[:, : self.V])
        best, at = self._scores.view(self.B, self._chunks, self._CHUNK).max(-1)
        chunk = best.argmax(-1, keepdim=True)
        return (chunk * self._CHUNK + at.gather(1, chunk)).squeeze(-1)

    def _step_logits(self) -> torch.Tensor:
        """One decode forward: ``[B, V]`` fp32 logits after the tokens in
        ``self.cur``, whose keys and values join the cache."""
        w, eps, dt = self._w, self.cfg.layer_norm_epsilon, self.dtype
        B, nh, dh, E = self.B, self.nh, self.dh, self.E
        cache = self.cache
        cache.extend(self.active)
        x = (w["wte"].index_select(0, self.cur)
             + w["wpe"].index_select(0, cache.start.clamp(max=self.T - 1)))

        def norm(x, name):
            return F.layer_norm(x.float(), (E,), w[f"{name[0]}_w{name[1]}"],
                                w[f"{name[0]}_b{name[1]}"], eps).to(dt)

        for i in range(self.L):
            qkv = torch.addmm(w[f"attn_b{i}"], norm(x, ("ln1", i)), w[f"attn_w{i}"])
            q, k, v = (t.view(B, 1, nh, dh) for t in qkv.split(E, dim=-1))
            cache.append(i, k, v, lengths=self.active)
            o = cache.attend(i, q[:, 0]).view(B, E)
            x = x + torch.addmm(w[f"proj_b{i}"], o, w[f"proj_w{i}"])
            h = torch.addmm(w[f"fc_b{i}"], norm(x, ("ln2", i)), w[f"fc_w{i}"])
            h = F.gelu(h, approximate="tanh")
            x = x + torch.addmm(w[f"fc2_b{i}"], h, w[f"fc2_w{i}"])
        xn = F.layer_norm(x.float(), (E,), w["lnf_w"], w["lnf_b"], eps)
        return torch.matmul(xn.to(dt), w["wte"].t()).float()

    def _sample(self, logits: torch.Tensor) -> None:
        """Sample the next token of every sequence and record it; stopped
        sequences record the end token outside the mask."""
        on = self.active.bool()
        nxt = self._draw(logits)
        if self.eos_token_id is not None:
            nxt = torch.where(on, nxt, self.eos_token_id)
        lp = ops.token_log_probs(logits, torch.where(on, nxt, -100), temperature=self.temperature)
        self.gen_buf.index_copy_(1, self.pos_out, nxt[:, None])
        self.lp_buf.index_copy_(1, self.pos_out, lp[:, None])
        self.mask_buf.index_copy_(1, self.pos_out, on[:, None])
        self.cur.copy_(nxt)
        if self.eos_token_id is not None:
            self.active.mul_(nxt != self.eos_token_id)
        self.pos_out.add_(1)

    def _decode_body(self) -> None:
        self._sample(self._step_logits())

    def capture(self) -> bool:
        # its warm-up decodes three tokens past the first
        return self.T >= 4 and super().capture()

    def prefill(self, prompts: torch.Tensor, lengths: Optional[torch.Tensor] = None) -> None:
        """HF forward over right-padded ``prompts [B, P]``; fills the cache
        with each sequence's first ``lengths`` positions (default: all) and
        samples the first response token."""
        B, P = prompts.shape
        if B != self.B or not 0 < P <= self.T:
            raise ValueError(f"PagedGPT2Decoder: prompts must be [{self.B}, up to {self.T}], got {list(prompts.shape)}")
        if lengths is None:
            lengths = torch.full((B,), P, dtype=torch.long)
        host = lengths.tolist()
        if len(host) != B or min(host) < 1 or max(host) > P:
            raise ValueError(f"PagedGPT2Decoder: lengths must hold {B} numbers from 1 to {P}, got {host}")
        self.cache.reset()
        self.cache.reserve([self.T] * B)
        count = lengths.to(device=self.device, dtype=torch.int32)
        # the decode step has no dropout, so the prompt gets none either
        training = [m for m in self._tr.modules() if m.training]
        try:
            for m in training:
                m.training = False
            with torch.no_grad(), torch.autocast(
                "cuda", dtype=self.dtype, cache_enabled=False, enabled=prompts.is_cuda,
            ):
                out = self._tr(input_ids=prompts, use_cache=True)
                last = out.last_hidden_state[torch.arange(B, device=prompts.device), count.long() - 1]
                logits = self.model.lm_head(last).float()
        finally:
            for m in training:
                m.training = True
        past = out.past_key_values
        self.cache.extend(count)
        with torch.no_grad():
            for i in range(self.L):
                if hasattr(past, "layers"):  # transformers >= 4.54 Cache
                    k, v = past.layers[i].keys, past.layers[i].values
                elif hasattr(past, "key_cache"):
                    k, v = past.key_cache[i], past.value_cache[i]
                else:
                    k, v = past[i]
                self.cache.append(i, k.transpose(1, 2).to(self.dtype),
                                  v.transpose(1, 2).to(self.dtype), lengths=count)
            self.active.fill_(1)
            self.mask_buf.fill_(False)
            self.lp_buf.zero_()
            self.pos_out.zero_()
            self._sample(logits)

    def rollout(self, prompts: torch.Tensor, gen_tokens: int,
                lengths: Optional[torch.Tensor] = None) -> TensorDict:
        """Generate up to ``gen_tokens`` tokens for each prompt.  Returns the
        keys the policy losses read: ``tokens_response``, ``log_probs`` (of
        the sampling distribution) and ``attention_mask_response``, all
        ``[B, gen_tokens]``."""
        if gen_tokens < 1 or prompts.shape[1] + gen_tokens > self.T:
            raise ValueError(
                f"PagedGPT2Decoder: {prompts.shape[1]} prompt and {gen_tokens} new tokens do not fit max_len {self.T}")
        self.prefill(prompts, lengths)
        with torch.no_grad():
            for _ in range(gen_tokens - 1):
                if self._graph is not None:
                    self._graph.replay()
                else:
                    self._decode_body()
        return TensorDict(
            {
                "tokens_response": self.gen_buf[:, :gen_tokens].clone(),
                "log_probs": self.lp_buf[:, :gen_tokens].clone(),
                "attention_mask_response": self.mask_buf[:, :gen_tokens].clone(),
            },
            batch_size=[self.B],
        )
