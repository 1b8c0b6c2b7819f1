"""BERT pretraining model (MLM + NSP heads), self-contained.

Capability parity with the reference's BERT benchmark path
(dear/bert_benchmark.py:72-112: transformers-2.11 BertForPreTraining built
from bert_config.json + BertPretrainingCriterion).  Configs: Base 12L/768h/12
heads, Large 24L/1024h/16 heads, vocab padded to a multiple of 8 (30528).
Attention runs through torch.nn.functional.scaled_dot_product_attention
(MIOpen/CK fused path on ROCm).

BertConfig(fused_ln=True) takes ops/fused_ln.py for every layer norm, with the
residual add in it; BertPretrainingCriterion(fused=True) takes the masked-token
loss from ops/token_loss.py, and BertDistillationCriterion adds what a teacher
says to it.  State dicts are the same either way."""
from dataclasses import dataclass

import torch
import torch.nn as nn
import torch.nn.functional as F

from ..ops.fused_ln import FusedLayerNorm
from ..ops.token_loss import (MAX_TOP, TokenLogProbs, token_logprobs,
                              topk_distill_loss)

__all__ = ["BertConfig", "BertForPreTraining", "BertPretrainingCriterion",
           "BertDistillationCriterion", "bert_base", "bert_large"]


@dataclass
class BertConfig:
    vocab_size: int = 30528          # 30522 padded %8 (reference :77-78)
    hidden_size: int = 768
    num_hidden_layers: int = 12
    num_attention_heads: int = 12
    intermediate_size: int = 3072
    max_position_embeddings: int = 512
    type_vocab_size: int = 2
    hidden_dropout_prob: float = 0.1
    attention_probs_dropout_prob: float = 0.1
    layer_norm_eps: float = 1e-12
    fused_ln: bool = False           # residual add + layer norm in one kernel


def _layer_norm(c: BertConfig):
    kind = FusedLayerNorm if c.fused_ln else nn.LayerNorm
    return kind(c.hidden_size, eps=c.layer_norm_eps)


def _add_norm(ln, x, h):
    """ln(x + h), the residual add inside of the kernel where it can be."""
    if isinstance(ln, FusedLayerNorm):
        return ln(h, residual=x)
    return ln(x + h)


def bert_base():
    return BertConfig()


def bert_large():
    return BertConfig(hidden_size=1024, num_hidden_layers=24,
                      num_attention_heads=16, intermediate_size=4096)


class BertEmbeddings(nn.Module):
    def __init__(self, c: BertConfig):
        super().__init__()
        self.word = nn.Embedding(c.vocab_size, c.hidden_size)
        self.position = nn.Embedding(c.max_position_embeddings, c.hidden_size)
        self.token_type = nn.Embedding(c.type_vocab_size, c.hidden_size)
        self.ln = _layer_norm(c)
        self.drop = nn.Dropout(c.hidden_dropout_prob)
        self.register_buffer("pos_ids",
                             torch.arange(c.max_position_embeddings)[None],
                             persistent=False)

    def forward(self, input_ids, token_type_ids):
        s = input_ids.size(1)
        e = self.word(input_ids) + self.position(self.pos_ids[:, :s]) \
            + self.token_type(token_type_ids)
        return self.drop(self.ln(e))


class BertSelfAttention(nn.Module):
    def __init__(self, c: BertConfig):
        super().__init__()
        self.nh = c.num_attention_heads
        self.hd = c.hidden_size // c.num_attention_heads
        self.qkv = nn.Linear(c.hidden_size, 3 * c.hidden_size)
        self.out = nn.Linear(c.hidden_size, c.hidden_size)
        self.p_drop = c.attention_probs_dropout_prob

    def forward(self, x, attn_mask):
        B, S, H = x.shape
        qkv = self.qkv(x).view(B, S, 3, self.nh, self.hd)
        q, k, v = (qkv[:, :, i].transpose(1, 2) for i in range(3))
        o = F.scaled_dot_product_attention(
            q, k, v, attn_mask=attn_mask,
            dropout_p=self.p_drop if self.training else 0.0)
        return self.out(o.transpose(1, 2).reshape(B, S, H))


class BertLayer(nn.Module):
    def __init__(self, c: BertConfig):
        super().__init__()
        self.attn = BertSelfAttention(c)
        self.ln1 = _layer_norm(c)
        self.fc1 = nn.Linear(c.hidden_size, c.intermediate_size)
        self.fc2 = nn.Linear(c.intermediate_size, c.hidden_size)
        self.ln2 = _layer_norm(c)
        self.drop = nn.Dropout(c.hidden_dropout_prob)

    def forward(self, x, attn_mask):
        x = _add_norm(self.ln1, x, self.drop(self.attn(x, attn_mask)))
        h = self.fc2(F.gelu(self.fc1(x)))
        return _add_norm(self.ln2, x, self.drop(h))


class BertModel(nn.Module):
    def __init__(self, c: BertConfig):
        super().__init__()
        self.embeddings = BertEmbeddings(c)
        self.layers = nn.ModuleList(BertLayer(c) for _ in range(c.num_hidden_layers))
        self.pooler = nn.Linear(c.hidden_size, c.hidden_size)

    def forward(self, input_ids, token_type_ids, attention_mask=None):
        mask = None
        if attention_mask is not None:
            mask = (attention_mask[:, None, None, :].to(torch.bool))
        x = self.embeddings(input_ids, token_type_ids)
        for layer in self.layers:
            x = layer(x, mask)
        pooled = torch.tanh(self.pooler(x[:, 0]))
        return x, pooled


class BertForPreTraining(nn.Module):
    """Sequence output -> tied-embedding MLM head; pooled -> NSP head."""

    def __init__(self, c: BertConfig):
        super().__init__()
        self.config = c
        self.bert = BertModel(c)
        self.transform = nn.Linear(c.hidden_size, c.hidden_size)
        self.transform_ln = _layer_norm(c)
        self.decoder = nn.Linear(c.hidden_size, c.vocab_size, bias=True)
        self.decoder.weight = self.bert.embeddings.word.weight  # tied
        self.nsp = nn.Linear(c.hidden_size, 2)
        self.apply(self._init)

    def _init(self, m):
        if isinstance(m, (nn.Linear, nn.Embedding)):
            nn.init.normal_(m.weight, std=0.02)
            if isinstance(m, nn.Linear) and m.bias is not None:
                nn.init.zeros_(m.bias)

    def forward(self, input_ids, token_type_ids, attention_mask=None):
        seq, pooled = self.bert(input_ids, token_type_ids, attention_mask)
        h = self.transform_ln(F.gelu(self.transform(seq)))
        return self.decoder(h), self.nsp(pooled)


class BertPretrainingCriterion(nn.Module):
    """MLM + NSP cross-entropy (reference dear/bert_benchmark.py:101-112).

    fused=True takes the MLM part from token_logprobs, which reads the logits
    of labelled tokens only."""

    def __init__(self, vocab_size, fused=False):
        super().__init__()
        self.vocab_size = vocab_size
        self.fused = fused
        self.ce = nn.CrossEntropyLoss(ignore_index=-1)

    def masked_token_loss(self, pred_scores, mlm_labels):
        """Mean over the labelled tokens; NaN where there is none, as
        nn.CrossEntropyLoss gives it."""
        scores = pred_scores.view(-1, self.vocab_size)
        labels = mlm_labels.view(-1)
        if not self.fused:
            return self.ce(scores, labels)
        lp = token_logprobs(scores, labels, ignore_index=-1).logprob
        return -lp.sum() / (labels != -1).sum()

    def forward(self, pred_scores, nsp_scores, mlm_labels, nsp_labels):
        mlm = self.masked_token_loss(pred_scores, mlm_labels)
        nsp = self.ce(nsp_scores.view(-1, 2), nsp_labels.view(-1))
        return mlm + nsp


class BertDistillationCriterion(BertPretrainingCriterion):
    """The pretraining loss of a student with a teacher's answers in it:

        (1 - weight) * MLM + weight * distillation + NSP

    The distillation part is the mean of topk_distill_loss over the labelled
    tokens, from the teacher's ``top`` alternatives at ``temperature``; with
    ``tail`` the rest of the vocabulary counts as one more alternative.
    """

    def __init__(self, vocab_size, top=32, temperature=1.0, weight=0.5,
                 tail=True):
        super().__init__(vocab_size, fused=True)
        if not 0.0 <= weight <= 1.0:
            raise ValueError(f"weight must be 0 to 1, got {weight}")
        if not 1 <= top <= min(MAX_TOP, vocab_size):
            raise ValueError(f"top must be 1 to {MAX_TOP} and at most the "
                             f"vocabulary, got {top}")
        self.top, self.temperature = top, temperature
        self.weight, self.tail = weight, tail

    @torch.no_grad()
    def answers(self, teacher_scores, mlm_labels) -> TokenLogProbs:
        """What the teacher says about the labelled tokens: this, not its
        logits, is kept or sent until the student's step."""
        return token_logprobs(teacher_scores, mlm_labels, top=self.top,
                              temperature=self.temperature, ignore_index=-1)

    def forward(self, pred_scores, nsp_scores, mlm_labels, nsp_labels,
                answers: TokenLogProbs):
        loss = topk_distill_loss(
            pred_scores, answers.top_ids, answers.top_logprobs,
            temperature=self.temperature, tail=self.tail)
        learned = loss.sum() / (mlm_labels != -1).sum()
        mlm = self.masked_token_loss(pred_scores, mlm_labels)
        nsp = self.ce(nsp_scores.view(-1, 2), nsp_labels.view(-1))
        return (1.0 - self.weight) * mlm + self.weight * learned + nsp
