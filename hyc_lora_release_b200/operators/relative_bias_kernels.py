"""Softmax of attention scores with a learned bias per bucket of relative positions, and its backward pass, for layers that know
positions by a bias on their scores instead of a rotation (no counterpart in the reference; beside ``softmax_kernels``)."""
import torch

from .._lib import host


class RelativeBuckets:
    """How distances share entries of a bias table: made once per model, given to the two functions below.

    One side has ``side = num_buckets // 2`` buckets if ``bidirectional`` (keys behind the query use the table's first half, keys
    ahead of it the second), else all ``num_buckets`` of them for keys behind (keys ahead use entry 0).  Distance r falls into bucket
    r for r < exact = side // 2, and into ``exact + floor((side - exact) * log(r / exact) / log(max_distance / exact))`` above, at
    most the last one.  The edges between buckets are found in whole numbers: no rounding decides a border.

    ``edges``: int32 [side] on the host, the smallest distance of each bucket."""
    __slots__ = ("num_buckets", "max_distance", "bidirectional", "edges")

    def __init__(self, num_buckets=32, max_distance=128, bidirectional=True):
        side = num_buckets // 2 if bidirectional else num_buckets
        if num_buckets < 2 or (bidirectional and num_buckets % 2) or not 2 <= side <= 128:
            raise ValueError("num_buckets must give 2 to 128 buckets per side, got %d (bidirectional: %s)" % (num_buckets, bidirectional))
        exact = side // 2
        rest = side - exact
        if not exact < max_distance <= 8192:
            raise ValueError("max_distance must be above %d and at most 8192, got %d" % (exact, max_distance))
        edges = list(range(exact))
        for t in range(rest):
            # the smallest r with rest * log(r / exact) >= t * log(max_distance / exact)
            bound, low, high = exact ** (rest - t) * max_distance ** t, exact, max_distance
            while low < high:
                r = (low + high) // 2
                if r ** rest >= bound:
                    high = r
                else:
                    low = r + 1
            edges.append(low)
        self.num_buckets, self.max_distance, self.bidirectional = num_buckets, max_distance, bool(bidirectional)
        self.edges = torch.tensor(edges, dtype=torch.int32, device="cpu")


def softmax_forward_relative_bias(scores, scale, table, buckets, attention_mask=None, causal=False, q_offset=0, inplace=False):
    """-> a = softmax(scores * scale + bias + attention_mask, dim=-1) in one pass, bias[i, j] = table[bucket(j - i - q_offset)] per head.

    scores [b, h, n, S] bf16, fp16 or fp32, S up to 131072; table [num_buckets, h] and the additive attention_mask
    [b or 1, h or 1, n or 1, S] each of one of these types; buckets: a ``RelativeBuckets``.  q_offset: position of the first row among
    the columns (S - n for queries at the end of a cache; a single token is n = 1).  causal: row i sees columns up to i + q_offset;
    what lies behind is not read and is 0 in the result.  A row that sees nothing (no column, or -infinity everywhere) is 0; where the
    mask is the type's lowest value instead, it shares its 1 among the columns, as the sum says: values up to the ends of a type's range are
    numbers like others, in scores, table and mask.  fp32 inside, rounded once.
    ``inplace`` overwrites ``scores`` (which must then be contiguous) and returns them."""
    return host.softmax_relative_bias_forward(scores, float(scale), table, buckets.edges, buckets.bidirectional, attention_mask, bool(causal),
                                              int(q_offset), bool(inplace))


def softmax_backward_relative_bias(a, grad_a, scale, buckets, causal=False, q_offset=0):
    """-> (grad_scores, grad_table) for the probabilities ``a`` and their gradient: ``ds = a * (grad_a - rowsum(a * grad_a))``,
    grad_scores = ds * scale in the type of ``a``, grad_table fp32 [num_buckets, h] = ds summed over batch, rows and the distances of a
    bucket, in a fixed order, rows that lie behind the last column (causal, i + q_offset >= S) among them.  ``scale``, ``buckets``, ``causal`` and ``q_offset`` as forward had them."""
    return host.softmax_relative_bias_backward(a, grad_a, float(scale), buckets.edges, buckets.bidirectional, bool(causal), int(q_offset))
