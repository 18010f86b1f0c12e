"""Attention modules with the reference's interface (layers/attention.py there).

MHA: fused QKV GEMM -> head-strided attention kernel (reads q/k/v as column slices of the QKV
buffer, writes the merged-head layout) -> output-projection GEMM.  None of the reference's five
rearrange copies is materialised.
ConvAttention (CvT): q/k/v GEMMs, depthwise 3x3 convolution of K and V directly on token-major
activations, attention with Skv != Sq, output projection.
"""
import torch
import torch.nn as nn

from .. import ops
from .dropout import Dropout
from .norm import QKNorm  # noqa: F401  (import parity with the reference module)


class MHA(nn.Module):
	def __init__(self, config):
		super().__init__()
		self.d_model = config.d_model
		self.n_head = config.n_head
		self.d_head = self.d_model // self.n_head
		if self.d_head * self.n_head != self.d_model:
			raise ValueError("d_model must be divisible by n_head")
		self.qkv_proj = nn.Linear(self.d_model, 3 * self.d_model, bias=False)
		self.out_proj = nn.Linear(self.d_model, self.d_model)
		self.dropout = Dropout(config.dropout)
		self.use_qk_norm = getattr(config, "use_qk_norm", False)
		if self.use_qk_norm:
			raise NotImplementedError("use_qk_norm=True is not supported (the reference's QKNorm cannot be constructed by its MHA either)")

	def forward(self, query):
		# dropout_p=self.dropout.p if self.training else 0.0 (layers/attention.py:41 there)
		drop = (self.dropout.p, ops.next_dropout_seed()) if self.dropout.active() else (0.0, 0)
		return ops.MHAFn.apply(query, self.qkv_proj.weight, self.out_proj.weight, self.out_proj.bias, self.n_head, drop)


class RelativeMHA(nn.Module):
	"""Multi-head self-attention with a learned relative position bias: a table entry per head for every (dy, dx) of the token grid (the
	*relative* attention of conv + attention hybrids), or per logarithmic bucket of the token distance.  Use as `config.attention`.

	config: d_model, n_head and MHA's keys (`qkv_proj`, `out_proj`), plus
	  attn_grid = (h, w)            one bucket per offset of an h x w grid of row-major tokens, or
	  attn_buckets = (n, far)       n buckets of the 1-D distance, logarithmic up to `far` (RelativeBuckets.log_distance); neither: no bias
	  n_kv_head                     key / value heads, a divisor of n_head (default n_head)
	  attn_softcap                  scores capped at +-softcap by a tanh (default 0: none)
	The table (`rel_bias`, [buckets, n_head]) starts at a normal distribution of 0.02; it is trained up to 8192 buckets (a grid of 45 x 45), larger
	ones evaluate only, or with the table frozen.  Attention-probability dropout is not supported."""

	def __init__(self, config):
		super().__init__()
		self.d_model, self.n_head = config.d_model, config.n_head
		self.n_kv_head = getattr(config, "n_kv_head", None) or config.n_head
		self.d_head = self.d_model // self.n_head
		if self.d_head * self.n_head != self.d_model or self.n_head % self.n_kv_head:
			raise ValueError("d_model must be divisible by n_head, and n_head by n_kv_head")
		self.softcap = float(getattr(config, "attn_softcap", 0.0))
		self.qkv_proj = nn.Linear(self.d_model, self.d_model + 2 * self.n_kv_head * self.d_head, bias=False)
		self.out_proj = nn.Linear(self.d_model, self.d_model)
		self.dropout = Dropout(config.dropout)
		self.grid, self.log_buckets = getattr(config, "attn_grid", None), getattr(config, "attn_buckets", None)
		if self.grid is not None and self.log_buckets is not None:
			raise ValueError("attn_grid and attn_buckets are alternatives")
		n = (2 * self.grid[0] - 1) * (2 * self.grid[1] - 1) if self.grid is not None else self.log_buckets[0] if self.log_buckets is not None else 0
		self.rel_bias = nn.Parameter(0.02 * torch.randn(n, self.n_head)) if n else None
		self._buckets = None

	def buckets(self, device):
		"""The RelativeBuckets of the module (built once per device)."""
		if self.rel_bias is None:
			return None
		if self._buckets is None or self._buckets.lookup.device != device:
			make = ops.RelativeBuckets
			with torch.inference_mode(False):  # (they outlive the call: a training step behind an inference-mode one saves them for its backward)
				self._buckets = make.grid(*self.grid, device) if self.grid is not None else make.log_distance(*self.log_buckets, device)
		return self._buckets

	def forward(self, query, segments=None, causal=False, prefix=None):
		"""query [B, S, d_model].  segments: int32 [B, S], images packed behind one another attend within their own number (negative:
		padding, zero output before the projection); causal / prefix: see ops.biased_attention."""
		if self.dropout.active():
			raise NotImplementedError("RelativeMHA has no dropout on the attention probabilities: set config.dropout = 0")
		if self.grid is not None and query.shape[1] != self.grid[0] * self.grid[1]:
			raise ValueError(f"attn_grid {self.grid} needs {self.grid[0] * self.grid[1]} tokens, got {query.shape[1]}")
		params = (self.qkv_proj.weight, self.out_proj.weight, self.out_proj.bias, self.rel_bias)
		return ops.RelativeMHAFn.apply(query, *params, self.n_head, self.n_kv_head, self.softcap, self.buckets(query.device), segments, causal, prefix,
			ops._wants_grad(query, *params))


class ConvAttention(nn.Module):
	def __init__(self, dim, n_head, kernel_size=3, qkv_stride=1, padding=1, dropout=0.1):
		super().__init__()
		self.n_head = n_head
		self.dim = dim
		self.d_head = dim // n_head
		self.q_proj = nn.Linear(dim, dim)
		self.k_proj = nn.Linear(dim, dim)
		self.v_proj = nn.Linear(dim, dim)
		self.conv_proj_k = nn.Conv2d(dim, dim, kernel_size, stride=qkv_stride, padding=padding, groups=dim, bias=False)
		self.conv_proj_v = nn.Conv2d(dim, dim, kernel_size, stride=qkv_stride, padding=padding, groups=dim, bias=False)
		self.out_proj = nn.Linear(dim, dim)
		self.dropout = Dropout(dropout)
		self.kernel_size, self.qkv_stride, self.padding = kernel_size, qkv_stride, padding

	def forward(self, x, h, w):
		# dropout_p=self.dropout.p if self.training else 0.0 (layers/attention.py:86 there)
		drop = (self.dropout.p, ops.next_dropout_seed()) if self.dropout.active() else (0.0, 0)
		return ops.ConvAttentionFn.apply(x, self.q_proj.weight, self.q_proj.bias, self.k_proj.weight, self.k_proj.bias,
			self.v_proj.weight, self.v_proj.bias, self.conv_proj_k.weight, self.conv_proj_v.weight,
			self.out_proj.weight, self.out_proj.bias, (h, w, self.n_head, self.kernel_size, self.qkv_stride, self.padding, drop))


class QuadrangleAttention(nn.Module):
	"""Learned-quadrangle window attention of the reference (layers/attention.py:95-283 there).
	Out of scope of the MI355X hot path; the name exists so that configs and `isinstance` checks
	written against the reference import cleanly.  Select `attention = MHA` in the config."""

	def __init__(self, config, lambda_reg=1.0):
		super().__init__()
		raise NotImplementedError("QuadrangleAttention is not part of the MI355X hot path: set config.attention = MHA")
