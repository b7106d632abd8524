"""Text generation with a MambaStack in 8 bits: prompts, single tokens, drawing.

The serving form of ``block.MambaStack`` (RMSNorm, real, Euler): the residual
stream stays float32, every block's residual addition, norm and quantisation
are one kernel (``rms_norm_fp8``), the input, output and vocabulary
projections are block-scaled 8-bit products (``fp8_matmul``) on weights
quantised once, prompts run through the conv and scan kernels in their (B, D,
L) layout, single tokens through the step kernels (Mamba.step,
mamba/mamba1.py:339-355), and ``sample_tokens`` draws. x_proj and dt_proj stay
in the decoder's `dtype`: they are small, and feed exponentials.
"""
from __future__ import annotations

import torch

from .causal_conv1d import causal_conv1d_fn, causal_conv1d_update
from .fp8 import fp8_matmul, quantize_fp8
from .rms_norm import rms_norm_fp8
from .sampling import sample_tokens
from .selective_scan_cuda import selective_scan_fn, selective_state_update


class _Layer:
    """A MambaBlock's weights as the decoder reads them."""

    def __init__(self, block, dtype):
        quant = lambda w: quantize_fp8(w.detach().float())  # noqa: E731
        f32 = lambda w: w.detach().to(torch.float32, copy=True).contiguous()  # noqa: E731
        self.norm = f32(block.norm.weight)
        self.w_main, self.w_skip = quant(block.w_main), quant(block.w_skip)
        self.w_out = quant(block.w_out)
        self.w_x = torch.cat([block.w_r, block.w_B, block.w_C]).detach().to(dtype)
        self.w_dt = block.w_dt.detach().to(dtype, copy=True)
        self.conv_w, self.conv_b = f32(block.conv_w), f32(block.conv_b)
        self.A = -torch.exp(f32(block.A_log))
        self.D, self.dt_bias = f32(block.D), f32(block.dt_bias)
        self.rank, self.n = block.dt_rank, block.d_state
        self.inner, self.kw = block.d_inner, block.kw


class MambaDecoder:
    """Generation with the weights of a ``MambaStack`` (norm_type "rmsnorm").

    The weights are copied at construction. ``prefill`` and ``step`` return
    float32 logits (B, vocab) of the last position; the state they hand on is
    a list of (conv state, scan state) per layer, updated in place by ``step``.
    The token -1, ``sample_tokens``' answer for a row with nothing to draw, makes
    that row's logits and state NaN, from which nothing is drawn either: -1 from there on.
    """

    def __init__(self, stack, dtype=torch.bfloat16):
        if not isinstance(stack.norm, torch.nn.RMSNorm) or not all(
                b.use_norm and isinstance(b.norm, torch.nn.RMSNorm) for b in stack.layers):
            raise ValueError("MambaDecoder needs a stack with norm_type 'rmsnorm'")
        if not stack.embed.is_cuda:
            raise ValueError("MambaDecoder needs a stack on a CUDA device")
        self.dtype, self.eps = dtype, stack.norm.eps
        # one row more, of NaN: what the token -1 indexes
        self.embed = torch.cat([stack.embed.detach().float(),
                                stack.embed.new_full((1, stack.embed.shape[1]), float("nan"),
                                                     dtype=torch.float32)])
        self.layers = [_Layer(b, dtype) for b in stack.layers]
        self.norm = stack.norm.weight.detach().to(torch.float32, copy=True)
        self.head = quantize_fp8(stack.head.detach().float())

    def _normed(self, branch, h, weight):
        """8-bit norm of the residual stream with the last branch added."""
        if branch is None:
            return (*rms_norm_fp8(h, weight, eps=self.eps), h)
        return rms_norm_fp8(branch, weight, h, eps=self.eps)

    def _logits(self, branch, h):
        q, s, _ = self._normed(branch, h, self.norm)
        return fp8_matmul(q, s, *self.head, out_dtype=torch.float32)

    @torch.no_grad()
    def prefill(self, tokens, seq_lens=None):
        """tokens (B, L), L >= 1, right-padded to seq_lens (B,) int32 if given:
        logits of each row's last token, and the state after it. Lengths above L
        count as L, as in the conv and the scan; a row of length 0 has NaN logits and
        the state before any token, from which ``step`` can go on."""
        if tokens.ndim != 2 or tokens.shape[1] < 1:
            raise ValueError("tokens must have shape (B, L) with L >= 1")
        batch, length = tokens.shape
        if seq_lens is not None:
            if (seq_lens.shape != (batch,) or seq_lens.dtype != torch.int32
                    or seq_lens.device != self.embed.device):
                raise ValueError("seq_lens must be an int32 tensor of shape (B,) on the "
                                 "weights' device")
            lens = seq_lens.long().clamp(0, length)
        h = self.embed[tokens].view(batch * length, -1)
        branch, state = None, []
        for p in self.layers:
            q, s, h = self._normed(branch, h, p.norm)
            x = fp8_matmul(q, s, *p.w_main, out_dtype=self.dtype, channel_major_batch=batch)
            z = fp8_matmul(q, s, *p.w_skip, out_dtype=self.dtype, channel_major_batch=batch)
            u, conv = causal_conv1d_fn(x, p.conv_w, p.conv_b, seq_lens, return_final_state=True)
            if seq_lens is not None:  # the last inputs of each row, not of the padding
                at = lens[:, None] + torch.arange(1 - p.kw, 0, device=x.device)
                conv = x.gather(2, at.clamp(min=0)[:, None].expand(-1, p.inner, -1))
                conv = conv.masked_fill((at < 0)[:, None], 0.0)
            xp = torch.matmul(p.w_x, u)
            delta = torch.matmul(p.w_dt, xp[:, :p.rank])
            y, last = selective_scan_fn(
                u, delta, p.A, xp[:, p.rank:p.rank + p.n].contiguous(),
                xp[:, p.rank + p.n:].contiguous(), p.D, z, p.dt_bias, True, True,
                seq_lens=seq_lens)
            branch = fp8_matmul(*quantize_fp8(y, channel_major=True), *p.w_out,
                                out_dtype=self.dtype)
            state.append((conv, last))
        end = (torch.full((batch,), length, device=tokens.device) if seq_lens is None
               else lens.clamp(min=1))
        rows = torch.arange(batch, device=tokens.device) * length + end - 1
        logits = self._logits(branch[rows], h[rows])
        if seq_lens is not None:
            logits.masked_fill_((lens < 1)[:, None], float("nan"))
        return logits, state

    @torch.no_grad()
    def step(self, tokens, state):
        """One token (B,) for every row: logits; state is updated in place."""
        h, branch = self.embed[tokens], None
        for p, (conv, scan) in zip(self.layers, state):
            q, s, h = self._normed(branch, h, p.norm)
            x = fp8_matmul(q, s, *p.w_main, out_dtype=self.dtype)
            z = fp8_matmul(q, s, *p.w_skip, out_dtype=self.dtype)
            u = causal_conv1d_update(x, conv, p.conv_w, p.conv_b)
            xp = u @ p.w_x.t()
            delta = xp[:, :p.rank] @ p.w_dt.t()
            y = selective_state_update(scan, u, delta, p.A, xp[:, p.rank:p.rank + p.n],
                                       xp[:, p.rank + p.n:], p.D, z, p.dt_bias, True)
            branch = fp8_matmul(*quantize_fp8(y), *p.w_out, out_dtype=self.dtype)
        return self._logits(branch, h)

    @torch.no_grad()
    def generate(self, tokens, new_tokens, seq_lens=None, uniform=None, generator=None,
                 **sampling):
        """new_tokens further tokens (B, new_tokens) for prompts (B, L); -1 where
        a row has nothing to draw.

        uniform (B, new_tokens) float32 in [0, 1) fixes the draws; without it
        they come from `generator` (on the tokens' device). sampling:
        ``sample_tokens``' temperature, top_k, top_p, min_p."""
        batch = tokens.shape[0]
        if uniform is None:
            uniform = torch.rand(batch, new_tokens, generator=generator, device=tokens.device)
        if uniform.shape != (batch, new_tokens):
            raise ValueError("uniform must have shape (B, new_tokens)")
        out = torch.empty(batch, new_tokens, dtype=torch.int64, device=tokens.device)
        if new_tokens == 0:
            return out
        logits, state = self.prefill(tokens, seq_lens)
        for t in range(new_tokens):
            if t:
                logits = self.step(out[:, t - 1], state)
            out[:, t] = sample_tokens(logits, uniform[:, t], **sampling)
        return out
