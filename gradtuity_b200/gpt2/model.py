"""GPT-2-small with the reference's module tree, attribute names and state_dict keys
(gpt2/model.py:25-149): wte + wpe + N x (ln1, attn, ln2, mlp_fc1, mlp_fc2) + ln_f + tied LM head.

Differences are inside `GPT2Block.__call__` only: `linear(...).gelu()` is one GEMM with a fused
bias+GELU epilogue that also stores the pre-activation for the backward, and the two residual adds
ride in the epilogues of the attention output projection and of the second MLP layer.  Activation
checkpointing and dropout > 0 are not part of this build.
"""
from __future__ import annotations

from ..nn import CausalSelfAttention, Dropout, Embedding, LayerNorm, Linear, Module, PositionalEmbedding, TiedLMHead
from ..tensor import Tensor

GPT2_SMALL = {
    "vocab_size": 50257, "n_positions": 1024, "n_embd": 768, "n_layer": 12, "n_head": 12, "n_inner": 3072,
    "embd_pdrop": 0.1, "attn_pdrop": 0.1, "resid_pdrop": 0.1,
}


class GPT2Block(Module):
    """Pre-LN attention + residual, pre-LN MLP + residual (gpt2/model.py:38-83)."""

    def __init__(self, n_embd: int, n_head: int, n_inner: int, attn_pdrop: float = 0.0, resid_pdrop: float = 0.0) -> None:
        super().__init__()
        self.ln1 = LayerNorm(n_embd)
        self.attn = CausalSelfAttention(embed_dim=n_embd, num_heads=n_head, attn_pdrop=attn_pdrop, resid_pdrop=resid_pdrop)
        self.ln2 = LayerNorm(n_embd)
        self.mlp_fc1 = Linear(n_embd, n_inner)
        self.mlp_fc2 = Linear(n_inner, n_embd)

    def __call__(self, x: Tensor) -> Tensor:
        x = self.attn(self.ln1(x), residual=x)                   # x + attn(ln1(x)): the add rides in the output projection
        h = self.ln2(x)
        B, S, E = h.shape
        # x + fc2(gelu(fc1(ln2(x)))): bias + GELU, the residual add and the GELU backward all sit in GEMM epilogues
        return h.view((B * S, E)).mlp_gelu(self.mlp_fc1.weight, self.mlp_fc1.bias, self.mlp_fc2.weight, self.mlp_fc2.bias,
                                           residual=x)

    def parameters(self) -> list[Tensor]:
        params = []
        for m in (self.ln1, self.attn, self.ln2, self.mlp_fc1, self.mlp_fc2):
            params.extend(m.parameters())
        return params


class GPT2Small(Module):
    """input_ids (B, S), float-encoded token ids -> logits (B, S, vocab_size) (gpt2/model.py:86-149)."""

    def __init__(self, vocab_size: int = 50257, n_positions: int = 1024, n_embd: int = 768, n_layer: int = 12,
                 n_head: int = 12, n_inner: int | None = None, embd_pdrop: float = 0.1, attn_pdrop: float = 0.1,
                 resid_pdrop: float = 0.1, use_checkpoint: bool = False) -> None:
        super().__init__()
        if n_inner is None:
            n_inner = 4 * n_embd
        if use_checkpoint:
            raise NotImplementedError("activation checkpointing is not part of this build")
        self.vocab_size = vocab_size
        self.n_positions = n_positions
        self.n_embd = n_embd
        self.n_layer = n_layer
        self.n_head = n_head
        self.n_inner = n_inner
        self.use_checkpoint = use_checkpoint
        self.wte = Embedding(vocab_size, n_embd)
        self.wpe = PositionalEmbedding(n_positions, n_embd)
        self.drop = Dropout(p=embd_pdrop)
        self.blocks = [GPT2Block(n_embd, n_head, n_inner, attn_pdrop, resid_pdrop) for _ in range(n_layer)]
        self.ln_f = LayerNorm(n_embd)
        self.lm_head = TiedLMHead(self.wte)

    def hidden(self, input_ids: Tensor) -> Tensor:
        """The hidden states (B, S, n_embd) that the head reads."""
        B, S = input_ids.shape
        x = self.wte(input_ids).add(self.wpe(seq_len=S, batch_size=B, start_pos=0))
        x = self.drop(x)
        for block in self.blocks:
            x = block(x)
        return self.ln_f(x)

    def __call__(self, input_ids: Tensor) -> Tensor:
        return self.lm_head(self.hidden(input_ids))

    def loss(self, input_ids: Tensor, labels: Tensor, ignore_index: int = -100) -> Tensor:
        """Mean cross entropy against labels (B * S,), the logits never kept (TiedLMHead.cross_entropy)."""
        return self.lm_head.cross_entropy(self.hidden(input_ids), labels, ignore_index=ignore_index)

    def distillation_loss(self, input_ids: Tensor, teacher_ids: Tensor, teacher_logits: Tensor, temperature: float = 1.0) -> Tensor:
        """Mean distillation loss against a teacher's top logits, (B * S, top) each (TiedLMHead.topk_distillation)."""
        return self.lm_head.topk_distillation(self.hidden(input_ids), teacher_ids, teacher_logits, temperature=temperature)

    def parameters(self) -> list[Tensor]:
        params = []
        params.extend(self.wte.parameters())
        params.extend(self.wpe.parameters())
        for block in self.blocks:
            params.extend(block.parameters())
        params.extend(self.ln_f.parameters())
        return params
