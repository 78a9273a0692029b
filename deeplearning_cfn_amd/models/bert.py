"""BERT-base pretraining model (BASELINE.json config #4).

The reference era had no transformers; BASELINE.json adds BERT-base as
the transformer DP config ("transformer path, MFMA GEMM").  Built from
scratch on the same ops seam: Linear routes through the MFMA GEMM kernel,
LayerNorm/GELU through their HIP kernels when native is selected,
attention through torch SDPA (flash-style, memory-bound-safe in 288 GB).
Data-parallel only, per SURVEY.md §3.3 scope ruling.

Documents of a batch may be packed: with ``cu_seqlens`` the tokens are read
one row behind the other, document i being the tokens from cu_seqlens[i] to
cu_seqlens[i + 1].  A document sees only itself, its positions begin at 0,
and its first token is what the NSP head reads.
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch
import torch.nn as nn
import torch.nn.functional as F


@dataclass
class BertConfig:
    vocab_size: int = 30522
    hidden: int = 768
    layers: int = 12
    heads: int = 12
    intermediate: int = 3072
    max_seq: int = 512
    type_vocab: int = 2
    dropout: float = 0.0          # pretraining-benchmark default: off
    layer_norm_eps: float = 1e-12
    # scores fall off with distance (slope 2 ** (-8 (h + 1) / heads) of head
    # h, both ways) instead of a table of positions
    alibi: bool = False


class MFMALinear(nn.Linear):
    """Linear that dispatches to the MFMA GEMM kernel on bf16/GPU."""

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        from ..ops import functional as F_amd
        shape = x.shape
        y = F_amd.linear(x.reshape(-1, shape[-1]), self.weight, self.bias)
        return y.reshape(*shape[:-1], self.out_features)


class FusedLayerNorm(nn.LayerNorm):
    def forward(self, x: torch.Tensor) -> torch.Tensor:
        from ..ops import functional as F_amd
        if hasattr(F_amd, "layer_norm"):
            return F_amd.layer_norm(x, self.normalized_shape, self.weight,
                                    self.bias, self.eps)
        return super().forward(x)


class SelfAttention(nn.Module):
    def __init__(self, cfg: BertConfig):
        super().__init__()
        self.heads = cfg.heads
        self.dh = cfg.hidden // cfg.heads
        self.qkv = MFMALinear(cfg.hidden, 3 * cfg.hidden)
        self.proj = MFMALinear(cfg.hidden, cfg.hidden)

    def forward(self, x: torch.Tensor, cu_seqlens: torch.Tensor | None = None,
                slopes: torch.Tensor | None = None) -> torch.Tensor:
        if cu_seqlens is not None:              # x: [tokens, hidden]
            from ..ops import functional as F_amd
            qkv = self.qkv(x).view(-1, 3, self.heads, self.dh)
            o = F_amd.document_attention_qkv(
                qkv, cu_seqlens, scale=1.0 / math.sqrt(self.dh),
                slopes=slopes)
            return self.proj(o.reshape(x.shape))
        B, S, H = x.shape
        qkv = self.qkv(x).view(B, S, 3, self.heads, self.dh)
        q, k, v = (qkv[:, :, i].transpose(1, 2) for i in range(3))
        if q.is_cuda:
            # Fused flash-style CDNA4 kernel (attention.hip) when shapes
            # qualify; otherwise explicit batched-GEMM + fp32 softmax —
            # never Triton / multi-backend dispatch.
            from ..ops import functional as F_amd
            o = F_amd.attention(q.contiguous(), k.contiguous(),
                                v.contiguous(),
                                scale=1.0 / math.sqrt(self.dh))
        else:
            o = F.scaled_dot_product_attention(q, k, v)
        return self.proj(o.transpose(1, 2).reshape(B, S, H))


class Block(nn.Module):
    def __init__(self, cfg: BertConfig):
        super().__init__()
        self.attn = SelfAttention(cfg)
        self.ln1 = FusedLayerNorm(cfg.hidden, eps=cfg.layer_norm_eps)
        self.fc1 = MFMALinear(cfg.hidden, cfg.intermediate)
        self.fc2 = MFMALinear(cfg.intermediate, cfg.hidden)
        self.ln2 = FusedLayerNorm(cfg.hidden, eps=cfg.layer_norm_eps)

    def forward(self, x: torch.Tensor, cu_seqlens: torch.Tensor | None = None,
                slopes: torch.Tensor | None = None) -> torch.Tensor:
        from ..ops import functional as F_amd
        x = self.ln1(x + self.attn(x, cu_seqlens, slopes))
        h = self.fc1(x)
        h = F_amd.gelu(h) if hasattr(F_amd, "gelu") else F.gelu(h)
        return self.ln2(x + self.fc2(h))


class BertForPretraining(nn.Module):
    """Encoder + MLM head (+NSP head) — the classic pretrain benchmark."""

    def __init__(self, cfg: BertConfig):
        super().__init__()
        self.cfg = cfg
        # vocab padded to a multiple of 64 so the weight-tied MLM-head
        # GEMM meets the MFMA kernel's alignment gate;
        # pad rows are never labeled, CE simply learns them away
        self.vocab_padded = (cfg.vocab_size + 63) // 64 * 64
        self.tok = nn.Embedding(self.vocab_padded, cfg.hidden)
        if cfg.alibi:
            slopes = torch.tensor([2.0 ** (-8.0 * (h + 1) / cfg.heads)
                                   for h in range(cfg.heads)])
            # as integers: a change of the model's type leaves them alone
            self.register_buffer("slope_bits", slopes.view(torch.int32),
                                 persistent=False)
        else:
            self.pos = nn.Embedding(cfg.max_seq, cfg.hidden)
        self.typ = nn.Embedding(cfg.type_vocab, cfg.hidden)
        self.ln = FusedLayerNorm(cfg.hidden, eps=cfg.layer_norm_eps)
        self.blocks = nn.ModuleList(Block(cfg) for _ in range(cfg.layers))
        self.mlm_dense = MFMALinear(cfg.hidden, cfg.hidden)
        self.mlm_ln = FusedLayerNorm(cfg.hidden, eps=cfg.layer_norm_eps)
        self.nsp = MFMALinear(cfg.hidden, 2)
        self.apply(self._init)

    @staticmethod
    def _init(m: nn.Module) -> None:
        if isinstance(m, (nn.Linear, nn.Embedding)):
            nn.init.normal_(m.weight, std=0.02)
            if isinstance(m, nn.Linear) and m.bias is not None:
                nn.init.zeros_(m.bias)

    def encode_documents(self, input_ids: torch.Tensor,
                         cu_seqlens: torch.Tensor,
                         token_type: torch.Tensor | None = None
                         ) -> torch.Tensor:
        """Packed documents: [*input_ids.shape, hidden].

        With a table of positions a document has at most ``max_seq`` tokens:
        the positions behind that are outside the table, which raises on the
        CPU and gives NaN for that document on the GPU (where the lengths are
        not known on the host).
        """
        from ..ops import functional as F_amd
        ids = input_ids.reshape(-1)
        # once, not in every layer; cut off at the tokens before it is narrowed
        cu = cu_seqlens.clamp(0, ids.numel()).to(torch.int32)
        typ = (token_type.reshape(-1) if token_type is not None
               else torch.zeros_like(ids))
        tables, index = [self.tok.weight, self.typ.weight], [ids, typ]
        slopes = None
        if self.cfg.alibi:
            slopes = self.slope_bits.view(torch.float32)
        else:
            tables.append(self.pos.weight)
            index.append(F_amd.document_positions(cu, ids.numel()))
        x = self.ln(F_amd.embedding_sum(index, tables))
        for blk in self.blocks:
            x = blk(x, cu, slopes)
        return x.view(*input_ids.shape, -1)

    def encode(self, input_ids: torch.Tensor,
               token_type: torch.Tensor | None = None,
               cu_seqlens: torch.Tensor | None = None) -> torch.Tensor:
        if self.cfg.alibi and cu_seqlens is None:
            n, S = input_ids.numel(), input_ids.shape[-1]
            cu_seqlens = torch.arange(0, n + 1, S, dtype=torch.int32,
                                      device=input_ids.device)
        if cu_seqlens is not None:
            return self.encode_documents(input_ids, cu_seqlens, token_type)
        B, S = input_ids.shape
        pos = torch.arange(S, device=input_ids.device).unsqueeze(0)
        typ = token_type if token_type is not None else torch.zeros_like(input_ids)
        x = self.ln(self.tok(input_ids) + self.pos(pos) + self.typ(typ))
        for blk in self.blocks:
            x = blk(x)
        return x

    def forward(self, input_ids: torch.Tensor,
                mlm_labels: torch.Tensor | None = None,
                nsp_labels: torch.Tensor | None = None,
                cu_seqlens: torch.Tensor | None = None):
        """``nsp_labels``: one a sequence, or one a document with
        ``cu_seqlens`` (-100 for an unused, empty one)."""
        x = self.encode(input_ids, cu_seqlens=cu_seqlens)
        h = self.mlm_ln(F.gelu(self.mlm_dense(x)))
        # MLM logits via weight tying with the token embedding; routed
        # through the MFMA GEMM (padded vocab keeps N % 16 == 0)
        from ..ops import functional as F_amd
        logits = F_amd.linear(h.reshape(-1, h.shape[-1]), self.tok.weight)
        logits = logits.reshape(*h.shape[:-1], self.vocab_padded)
        if mlm_labels is None:
            return logits
        loss = F.cross_entropy(
            logits.float().view(-1, self.vocab_padded),
            mlm_labels.view(-1), ignore_index=-100)
        if nsp_labels is not None:
            if cu_seqlens is None:
                first = x[:, 0]
            else:
                flat = x.reshape(-1, x.shape[-1])
                first = flat[cu_seqlens[:-1].long()
                             .clamp(0, flat.shape[0] - 1)]
            cls = self.nsp(first)
            loss = loss + F.cross_entropy(cls.float(), nsp_labels)
        return loss


def build_bert(size: str = "base", seq_len: int = 128,
               alibi: bool = False) -> BertForPretraining:
    if size == "base":
        cfg = BertConfig()
    elif size == "large":
        cfg = BertConfig(hidden=1024, layers=24, heads=16, intermediate=4096)
    else:
        raise ValueError(f"unknown bert size {size!r}")
    cfg.max_seq = max(cfg.max_seq, seq_len)
    cfg.alibi = alibi
    return BertForPretraining(cfg)
