"""Block LR-AttnRes GPT for the whole-model measurement.

A compact restatement of the reference model's forward (OBPM, model.py:735 and
its generic block path, model.py:2225-2620) for one family of settings:
`use_attnres` with block AttnRes (`attnres_type="block"`), LRID keys from the
fused output projections (`LRIDFusedProjection`, model.py:316-388, fused-key
layout), static depth queries, the block-count logit prior (legacy beta),
count / sqrt block averaging (legacy alpha), per-head key norm, rotary
embeddings, q/k norm, SwiGLU MLPs and RMS norms before or after each sublayer;
or, with `lrid_key_from_output_tail` (model.py:101, :377-378, :418-419), keys
that are the last `lrid_rank` columns of each source's value.
Module and parameter names follow the reference, so a reference state_dict
loads into it (tests/test_gpt_model.py checks the forward against OBPM).

`fused=True` routes every depth read and block summary through this package's
kernels (`lrid_attention_residual_read`, `attention_residual_block_summary`,
`lrid_fused_projection_forward`); `fused=False` uses the reference's PyTorch
read (model.py:2130-2159) -- the model's unfused path. Everything else
(attention, GEMMs) is PyTorch.

`fused_layer=True` (16-bit models) also runs the layer around the reads on this
package's operators: the q/k norm with the rotation and the split into heads as
one kernel (`qk_norm_rope`) and the MLP up to its output projection as another
(`swiglu_projection`), in training and inference.

`GPT.generate` continues prompts greedily over a `GPTCache`: keys and values of
every layer in 4-bit pages (`kv4_append`), attended to by the new tokens
(`kv4_attention`). A prompt itself is attended to in full precision while it is
written.
"""
import math
from dataclasses import dataclass
from typing import Optional

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch import Tensor


@dataclass
class GPTConfig:
    n_layer: int = 24
    n_head: int = 16
    n_embd: int = 1024
    mlp_hidden_dim: Optional[int] = None  # default n_embd * 4 (model.py:574)
    vocab_size: int = 100277
    block_size: int = 2048
    rope_theta: float = 500000.0
    norm_pos: str = "after"
    qk_norm: bool = True
    init_std: float = 0.02
    attnres_num_blocks: int = 12
    attnres_block_average_mode: str = "count"
    attnres_block_count_prior: bool = True
    attnres_key_norm: bool = True
    attnres_fuse_read_norm: bool = True
    lrid_rank: int = 64
    lrid_num_heads: int = 2
    lrid_key_from_output_tail: bool = False
    pad_vocab_to: int = 64
    attn_res_query_init: str = "zero"
    fused: bool = True
    fused_layer: bool = False

    @property
    def hidden_dim(self) -> int:
        return self.mlp_hidden_dim if self.mlp_hidden_dim is not None else int(self.n_embd * 4)

    @property
    def lrid_logit_scale(self) -> float:
        return 1.0 / math.sqrt(self.lrid_rank // self.lrid_num_heads)  # model.py:203-205


def norm(x: Tensor) -> Tensor:
    return F.rms_norm(x, (x.size(-1),))


def norm_heads(x: Tensor, heads: int) -> Tensor:
    """Per-head RMS norm of the last dim (model.py:34-37)."""
    s = x.shape
    return norm(x.reshape(*s[:-1], heads, s[-1] // heads)).reshape(s)


class RotaryEmbedding(nn.Module):
    def __init__(self, cfg: GPTConfig):
        super().__init__()
        self.cfg = cfg
        cos, sin = self._angles()
        self.register_buffer("sin", sin[None, None])
        self.register_buffer("cos", cos[None, None])
        self._exact = cos.float().clone(), sin.float().clone()
        self._made = None

    def _angles(self, device=None):
        """Cosines and sines [block_size, head_dim / 2] of the config."""
        dim = self.cfg.n_embd // self.cfg.n_head
        inv_freq = 1.0 / (self.cfg.rope_theta ** (torch.arange(0, dim, 2, device=device) / dim))
        freq = torch.outer(torch.arange(self.cfg.block_size, device=device), inv_freq)
        return freq.cos(), freq.sin()

    @property
    def tables(self):
        """Cosines and sines as qk_norm_rope takes them: [block_size, head_dim / 2] float32 on the module's device, of
        the values that its cos and sin buffers hold. Made again when a buffer was replaced or written to."""
        buffers = self.cos, self.sin
        if torch.compiler.is_compiling():
            return self._follow(buffers)
        versions = tuple(None if b.is_inference() else b._version for b in buffers)
        if self._made is not None:
            of, at, made = self._made
            if of[0] is buffers[0] and of[1] is buffers[1] and at == versions:
                return made
        made = self._follow(buffers)
        if made[0].is_cuda and type(made[0]) is Tensor:  # not a fake one, which no stream makes
            if torch.cuda.is_current_stream_capturing():
                return made  # the graph's own
            torch.cuda.current_stream(made[0].device).synchronize()  # any stream may use them next
        self._made = buffers, versions, made
        return made

    def _follow(self, buffers):
        """The buffers in float32. Where a 16-bit buffer holds the config's values rounded, the values (chosen on the
        device: nothing waits for it)."""
        device = buffers[0].device
        if self._exact[0].device != device and not torch.compiler.is_compiling():
            if self._exact[0].is_meta:  # the module was built without data
                self._exact = self._angles("cpu")
            self._exact = tuple(t.to(device, torch.float32) for t in self._exact)
        return tuple(b[0, 0] if b.dtype == torch.float32
                     else torch.where((b[0, 0] == e.to(b.dtype)).all(), e, b[0, 0].float())
                     for b, e in zip(buffers, self._exact))

    def _apply(self, fn, recurse=True):
        super()._apply(fn, recurse)
        self.tables  # made here rather than in the middle of a step
        return self

    def _load_from_state_dict(self, *args, **kwargs):
        super()._load_from_state_dict(*args, **kwargs)
        self.tables

    def rotate(self, x: Tensor) -> Tensor:
        T = x.size(-2)
        sin, cos = self.sin[:, :, :T], self.cos[:, :, :T]
        x1, x2 = x[..., 0::2], x[..., 1::2]
        return torch.stack([cos * x1 - sin * x2, sin * x1 + cos * x2], dim=-1).flatten(-2)


class LRIDFusedProjection(nn.Module):
    """Output projection emitting the sublayer output and its LRID key (the
    reference's fused-key layout: one weight [output + rank, input]; with the
    output-tail key, weight [output, input] and key = output[..., -rank:])."""

    def __init__(self, cfg: GPTConfig, input_dim: int, output_dim: int):
        super().__init__()
        self.cfg = cfg
        self.output_dim = output_dim
        extra = 0 if cfg.lrid_key_from_output_tail else cfg.lrid_rank
        self.proj = nn.Linear(input_dim, output_dim + extra, bias=False)

    def forward(self, x: Tensor):
        c = self.cfg
        if c.lrid_key_from_output_tail:
            out = self.proj(x)
            # the fused read takes the key as a strided view of the output rows;
            # the PyTorch path copies it like the reference (model.py:377-378)
            key = out[..., -c.lrid_rank:]
            return out, (key if c.fused else key.contiguous())
        if c.fused:
            from .ops import lrid_fused_projection_forward

            return lrid_fused_projection_forward(x, self.proj.weight, self.output_dim, c.lrid_rank, c.lrid_num_heads,
                                                 c.attnres_key_norm)
        y = self.proj(x)
        out = y[..., :self.output_dim].contiguous()
        key = y[..., self.output_dim:self.output_dim + c.lrid_rank]
        if c.attnres_key_norm:
            key = norm_heads(key, c.lrid_num_heads)
        return out, key


class LRIDSourceKeyProjection(nn.Module):
    """Key of the embedding source (model.py:391-423): proj(x), per-head normed,
    or the last `lrid_rank` columns of x with the output-tail key."""

    def __init__(self, cfg: GPTConfig):
        super().__init__()
        self.cfg = cfg
        self.proj = None if cfg.lrid_key_from_output_tail else nn.Linear(cfg.n_embd, cfg.lrid_rank, bias=False)

    def forward(self, x: Tensor) -> Tensor:
        if self.proj is None:
            key = x[..., -self.cfg.lrid_rank:]
            return key if self.cfg.fused else key.contiguous()
        key = self.proj(x)
        return norm_heads(key, self.cfg.lrid_num_heads) if self.cfg.attnres_key_norm else key


class MultiHeadAttention(nn.Module):
    def __init__(self, cfg: GPTConfig):
        super().__init__()
        self.cfg = cfg
        self.head_dim = cfg.n_embd // cfg.n_head
        self.rope = RotaryEmbedding(cfg)
        self.c_attn = nn.Linear(cfg.n_embd, 3 * cfg.n_embd, bias=False)
        self.c_proj = LRIDFusedProjection(cfg, cfg.n_embd, cfg.n_embd)

    def _heads(self, x: Tensor, positions: Optional[Tensor]):
        """Queries, keys and values [B, T, heads, head_dim], q and k normed and rotated."""
        from .layer import qk_norm_rope

        H = self.cfg.n_head
        return qk_norm_rope(self.c_attn(x), H, H, *self.rope.tables, positions=positions,
                            normalize=self.cfg.qk_norm)

    def forward(self, x: Tensor, past: Optional["LayerPast"] = None):
        B, T, C = x.shape
        if past is not None:
            return self.c_proj(past.attend(*self._heads(x, past.positions)).reshape(B, T, C))
        if self.cfg.fused_layer:
            q, k, v = (t.transpose(1, 2) for t in self._heads(x, None))
        else:
            q, k, v = self.c_attn(x).split(C, dim=2)
            q, k, v = (t.view(B, T, self.cfg.n_head, self.head_dim).transpose(1, 2) for t in (q, k, v))
            if self.cfg.qk_norm:
                q, k = norm(q), norm(k)
            q, k = self.rope.rotate(q), self.rope.rotate(k)
        y = F.scaled_dot_product_attention(q, k, v, is_causal=True)
        return self.c_proj(y.transpose(1, 2).contiguous().view(B, T, C))


class GPTCache:
    """Keys and values of `batch` sequences of up to `max_tokens` tokens for every layer of a GPT, in
    4 bits: one pool of pages a layer, one page table for all."""

    def __init__(self, cfg: GPTConfig, batch: int, max_tokens: int, page_size: int = 64, device="cuda"):
        from .layer import KV4Cache

        if max_tokens > cfg.block_size:
            raise RuntimeError(f"attnres_b200: GPTCache of {max_tokens} tokens, the model has {cfg.block_size} positions")
        per = -(-max_tokens // page_size)
        self.max_tokens, self.used = max_tokens, 0
        self.pools = [KV4Cache.empty(batch * per, page_size, cfg.n_head, cfg.n_embd // cfg.n_head, device)
                      for _ in range(cfg.n_layer)]
        self.page_table = torch.arange(batch * per, device=device, dtype=torch.int32).view(batch, per)
        self.lengths = torch.zeros(batch, device=device, dtype=torch.int32)

    def check_room(self, tokens: int):
        if self.used + tokens > self.max_tokens:
            raise RuntimeError(f"attnres_b200: the cache holds {self.used} of {self.max_tokens} tokens, {tokens} more do not fit")


class LayerPast:
    """What a layer's attention takes of a GPTCache for one call: new tokens are written behind the
    sequences' and attend to all of them (to each other alone, in full precision, while the cache is empty)."""

    def __init__(self, cache: GPTCache, layer: int, positions: Tensor, lengths: Tensor):
        self.cache, self.pool, self.positions, self.lengths = cache, cache.pools[layer], positions, lengths

    def attend(self, q: Tensor, k: Tensor, v: Tensor) -> Tensor:
        from .layer import kv4_append, kv4_attention

        kv4_append(self.pool, k, v, self.cache.page_table, self.cache.lengths)
        if self.cache.used == 0:
            q, k, v = (t.transpose(1, 2) for t in (q, k, v))
            return F.scaled_dot_product_attention(q, k, v, is_causal=True).transpose(1, 2)
        return kv4_attention(q, self.pool, self.cache.page_table, self.lengths)


class MLP(nn.Module):
    def __init__(self, cfg: GPTConfig):
        super().__init__()
        self.cfg = cfg
        self.fc1 = nn.Linear(cfg.n_embd, cfg.hidden_dim * 2, bias=False)
        self.fc2 = LRIDFusedProjection(cfg, cfg.hidden_dim, cfg.n_embd)

    def forward(self, x: Tensor):
        if self.cfg.fused_layer:
            from .layer import swiglu_projection

            return self.fc2(swiglu_projection(x, self.fc1.weight))
        x, gate = self.fc1(x).chunk(2, dim=-1)
        return self.fc2(F.silu(gate) * x)


class Block(nn.Module):
    def __init__(self, cfg: GPTConfig):
        super().__init__()
        self.cfg = cfg
        self.attn = MultiHeadAttention(cfg)
        self.mlp = MLP(cfg)

    def _sublayer(self, f, x: Tensor, x_is_normalized: bool, *args):
        if self.cfg.norm_pos == "before" and not x_is_normalized:
            x = norm(x)
        out, key = f(x, *args)
        if self.cfg.norm_pos == "after":
            out = norm(out)
        return out, key

    def forward_attention(self, x, x_is_normalized=False, past=None):
        return self._sublayer(self.attn, x, x_is_normalized, *(() if past is None else (past,)))

    def forward_mlp(self, x, x_is_normalized=False):
        return self._sublayer(self.mlp, x, x_is_normalized)


class GPT(nn.Module):
    """OBPM with block LR-AttnRes (see the module docstring)."""

    def __init__(self, cfg: GPTConfig):
        super().__init__()
        self.cfg = cfg
        H, dk = cfg.lrid_num_heads, cfg.lrid_rank // cfg.lrid_num_heads
        self.transformer = nn.ModuleDict(dict(
            wte=nn.Embedding(cfg.vocab_size, cfg.n_embd),
            layers=nn.ModuleList([Block(cfg) for _ in range(cfg.n_layer)]),
            lrid_embedding_key=LRIDSourceKeyProjection(cfg),
            lrid_queries=nn.ParameterList([nn.Parameter(torch.empty(H, dk)) for _ in range(2 * cfg.n_layer)]),
        ))
        self.lm_head = nn.Linear(cfg.n_embd, cfg.vocab_size, bias=False)
        total = 2 * cfg.n_layer
        nb = min(cfg.attnres_num_blocks, total)
        self.block_ends = frozenset(math.ceil(total * i / nb) for i in range(1, nb + 1))  # model.py:828-836
        for m in self.modules():
            if isinstance(m, (nn.Linear, nn.Embedding)):
                nn.init.normal_(m.weight, mean=0.0, std=cfg.init_std)
        for q in self.transformer.lrid_queries:
            if cfg.attn_res_query_init == "zero":
                nn.init.zeros_(q)
            else:
                nn.init.normal_(q, mean=0.0, std=cfg.init_std)

    # ---- block bookkeeping (model.py:955-1069) --------------------------------
    def _scale(self, count: int) -> float:
        alpha = 0.5 if self.cfg.attnres_block_average_mode == "sqrt" else 1.0
        return float(count) ** (-alpha)

    def _bias(self, count: int) -> float:
        return math.log(float(count)) if (self.cfg.attnres_block_count_prior and count != 1) else 0.0

    def _biases(self, counts):
        b = [self._bias(c) for c in counts]
        return b if any(v != 0.0 for v in b) else None

    def _summary(self, partial: Optional[Tensor], out: Tensor, count: int):
        """New running block sum and its block source value (sum * count^-alpha)."""
        if self.cfg.fused:
            from .ops import attention_residual_block_summary

            alpha = 0.5 if self.cfg.attnres_block_average_mode == "sqrt" else 1.0
            return attention_residual_block_summary(partial, out, count=count, alpha=alpha)
        s = out if partial is None else partial + out
        return s, s * self._scale(count)

    def _read(self, idx: int, values, keys, biases, normalize_output: bool) -> Tensor:
        """The depth read at residual site `idx` (model.py:2081-2159)."""
        if len(values) == 1:
            return norm(values[0]) if normalize_output else values[0]
        c = self.cfg
        query = self.transformer.lrid_queries[idx - 1]
        if c.fused:
            from .ops import lrid_attention_residual_read

            return lrid_attention_residual_read(values, keys, query, c.lrid_num_heads, c.lrid_logit_scale,
                                                c.attnres_key_norm, normalize_output=normalize_output,
                                                source_logit_biases=biases)
        from .torch_ref import lrid_attention_residual_read_torch

        out = lrid_attention_residual_read_torch(values, keys, query, c.lrid_num_heads, c.lrid_logit_scale,
                                                 c.attnres_key_norm, source_logit_biases=biases)
        return norm(out) if normalize_output else out

    def forward(self, idx: Tensor, return_hidden: bool = False, cache: Optional[GPTCache] = None) -> Tensor:
        """Logits [B, T, vocab] (or the normed hidden states). With a cache the tokens are the next
        ones of its sequences, and are in it afterwards (no gradient)."""
        c = self.cfg
        x = self.transformer.wte(idx)
        pasts = [None] * c.n_layer
        if cache is not None:
            T = idx.size(1)
            cache.check_room(T)
            if cache.used:
                self._check_cached_attention()
            positions = cache.lengths[:, None] + torch.arange(T, device=idx.device, dtype=torch.int32)
            lengths = cache.lengths + T
            pasts = [LayerPast(cache, li, positions, lengths) for li in range(c.n_layer)]
        fused_read_norm = (c.fused and c.norm_pos == "before" and c.attnres_fuse_read_norm
                           and c.lrid_num_heads == 1)  # model.py:2237-2243
        # completed block sources (value, key) and their counts; the live block
        done_v, done_k, done_n = [x], [self.transformer.lrid_embedding_key(x)], [1]
        part, part_src, part_key, part_n = None, None, None, 0

        def sources():
            if part is None:
                return done_v, done_k, done_n
            return done_v + [part_src], done_k + [part_key], done_n + [part_n]

        def read(site):
            v, k, n = sources()
            return self._read(site, v, k, self._biases(n), fused_read_norm)

        for li, block in enumerate(self.transformer.layers):
            for sub in (0, 1):
                site = 2 * li + sub
                x = read(site) if site > 0 else (norm(x) if fused_read_norm else x)
                f, past = ((block.forward_attention, pasts[li]), (block.forward_mlp, None))[sub]
                out, key = f(x, x_is_normalized=fused_read_norm, **({} if past is None else {"past": past}))
                part_n += 1
                part, part_src = self._summary(part, out, part_n)
                part_key = key if part_n == 1 else part_key + key
                if site + 1 in self.block_ends:
                    done_v.append(part_src)
                    done_k.append(part_key)
                    done_n.append(part_n)
                    part, part_src, part_key, part_n = None, None, None, 0
        x = read(2 * c.n_layer)
        if not fused_read_norm:
            x = norm(x)
        if cache is not None:
            cache.lengths = lengths
            cache.used += T
        return x if return_hidden else self.logits(x)

    def _check_cached_attention(self):
        """Raises where kv4_attention will not take the model's heads: better now than after the prompt's work."""
        c, weight = self.cfg, self.transformer.wte.weight
        dtype = torch.get_autocast_dtype(weight.device.type) if torch.is_autocast_enabled(weight.device.type) else weight.dtype
        head_dim = c.n_embd // c.n_head
        if dtype not in (torch.float16, torch.bfloat16) or head_dim not in (64, 128):
            raise RuntimeError("attnres_b200: tokens behind a cache's go through kv4_attention, which is built for float16 and "
                               f"bfloat16 and heads of 64 and 128, not for {dtype} and {head_dim}")

    @torch.no_grad()
    def generate(self, idx: Tensor, new_tokens: int, cache: Optional[GPTCache] = None) -> Tensor:
        """The prompts idx [B, T] with `new_tokens` tokens appended to each, the likeliest at every
        step. Pass a cache to go on from it later; the last token chosen is not in it yet."""
        if new_tokens < 1:
            return idx
        if new_tokens > 1 or (cache is not None and cache.used):
            self._check_cached_attention()
        if cache is None:
            cache = GPTCache(self.cfg, idx.size(0), idx.size(1) + new_tokens - 1, device=idx.device)
        cache.check_room(idx.size(1) + new_tokens - 1)
        out, step = [idx], idx
        for _ in range(new_tokens):
            step = self.logits(self(step, return_hidden=True, cache=cache)[:, -1:]).argmax(-1)
            out.append(step)
        return torch.cat(out, dim=1)

    def logits(self, x: Tensor) -> Tensor:
        """lm_head(x). With a vocabulary that is not a multiple of
        `pad_vocab_to` (the reference's 100 277 is odd) the logit rows are not
        16-byte aligned and the library GEMMs fall back to slow kernels, so
        the logits are computed against the weight padded with zero rows and
        returned as the [..., :vocab] view: the same values; the pad's backward
        drops the padding's gradient. Both read paths do this."""
        w = self.lm_head.weight
        pad = -w.size(0) % self.cfg.pad_vocab_to if self.cfg.pad_vocab_to > 1 else 0
        if pad == 0:
            return self.lm_head(x)
        return F.linear(x, F.pad(w, (0, 0, 0, pad)))[..., :w.size(0)]
