"""RMS norms of the query and key heads with the rotary embedding in the same pass, for layers that norm each head before the
scores (no counterpart in the reference, whose layers rotate what the projections give: ``rope_kernels``)."""
from .._lib import host


def qk_norm_rope_forward(q, k, q_weight, k_weight, cos, sin, eps, position_ids=None, rotary_dim=None):
    """-> (q_out, k_out), new contiguous tensors.  For every head x of ``q`` [batch, seq_len, heads, head_dim] and ``k``
    [batch, seq_len, kv_heads, head_dim]: ``n = x / sqrt(mean(x^2) + eps) * weight``, then the rotate-half embedding on the first
    ``rotary_dim`` channels (default: all), as ``rope_forward`` has it:
    ``out[j] = n[j] cos - n[j + rotary_dim / 2] sin``, ``out[j + rotary_dim / 2] = n[j + rotary_dim / 2] cos + n[j] sin``.
    Computed in fp32 and rounded once.

    q, k: one type of bf16, fp16, fp32; any strides (slices of a joint projection are read in place; what does not lie on 16 bytes
    is copied).  q_weight, k_weight: [head_dim], one type.  cos, sin: tables of [positions, >= rotary_dim / 2], of which the first
    rotary_dim / 2 columns are read.  position_ids: int32 or int64 [batch or 1, seq_len], default 0, 1, 2, ... in every sequence; a
    position that the tables do not have gives NaN in the rotated channels.  head_dim and rotary_dim are multiples of 16, head_dim
    at most 512."""
    return host.qk_norm_rope_forward(q, k, q_weight, k_weight, cos, sin, float(eps), position_ids, rotary_dim)


def qk_norm_rope_backward(dq, dk, q, k, q_weight, k_weight, cos, sin, eps, position_ids=None, rotary_dim=None, needs_weight_grad=True):
    """-> (grad_q, grad_k, grad_q_weight, grad_k_weight) for the gradients ``dq``, ``dk`` of ``qk_norm_rope_forward``'s results
    (any strides, expanded ones among them); q, k and the rest as forward took them.  The weights' gradients are summed in fp32 in a
    fixed order and returned in the weights' type; ``needs_weight_grad=False``: None for both (frozen norms)."""
    return host.qk_norm_rope_backward(dq, dk, q, k, q_weight, k_weight, cos, sin, float(eps), position_ids, rotary_dim, bool(needs_weight_grad))
