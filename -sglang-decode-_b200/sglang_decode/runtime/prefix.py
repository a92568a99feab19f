"""Decode of a batch whose requests share a prefix: the prefix's K and V are read once for all.

``SharedPrefixEngine`` is a ``DecodeEngine`` (the plan, the modes and ``prepare()`` are the same) whose
plan covers each request's OWN tokens, those after the prefix.  ``execute`` attends every request
to the prefix in one matrix product, decodes the own tokens as ``DecodeEngine`` does, and merges
both parts: the result is the decode of prefix + own tokens.  No counterpart in the reference.
"""
import torch

from .. import _native
from ..config import DecodeConfig
from .engine import DecodeEngine


def own_splits(lengths, config: DecodeConfig):
    """Split counts for the own tokens of a batch: enough tasks to give every worker four, no more.

    Own tokens are short next to the prefix, so that a fixed number of splits would cut them into
    many small tasks, each with a partial result to merge (256 requests of 576 tokens on average, 8
    KV heads: 230 us and 44 us of merge with up to 16 splits, 119 us and 34 us with these)."""
    tasks = sum(lengths) * config.kv_heads
    chunk = max(256, -(-tasks // (4 * config.workers)))
    return [max(1, min(config.max_splits, -(-n // chunk))) for n in lengths]


class SharedPrefixEngine(DecodeEngine):
    """``prefix_capacity``: the most prefix tokens an ``execute`` may name (a multiple of the page
    size).  The workspace for it is allocated here, once, for all layers: like the rest of an
    engine it serves one serial stream."""

    def __init__(self, config: DecodeConfig, prefix_capacity, device="cuda", dtype=torch.bfloat16, layers=1, rules=(),
                 force_mode=-1):
        if prefix_capacity < 0 or prefix_capacity % config.page_size:
            raise ValueError("prefix_capacity must be whole pages, 0 or more")
        super().__init__(config, device, dtype, layers, rules, force_mode)
        self.prefix_capacity = int(prefix_capacity)
        c = config
        size = _native.prefix_workspace_bytes(c.batch_capacity, c.query_heads, c.kv_heads, c.head_dim, self.prefix_capacity)
        self.workspace = torch.empty(size, dtype=torch.uint8, device=self.plan.device)
        self._decode_prefix = _native.op("decode_shared_prefix")

    def execute(self, q, k, v, pages, prefix, layer=0, *, prefix_length=None, indptr=None, scale=None, logit_cap=0.0,
                k_new=None, v_new=None, new_loc=None):
        """As ``DecodeEngine.execute``, with ``prefix`` (int32, on the GPU): the prefix's token slots
        for CSR KV, its pages for paged KV.

        ``prefix_length`` (int32[1] on the GPU; default: all that ``prefix`` names) lets a captured
        call follow a prefix whose length changes; lengths past what ``prefix`` names are cut to it.
        An index outside the pool reads as a zero row.  Requests without own tokens attend to the
        prefix alone; rows at or past the plan's active count are zero.  With CSR KV ``pages`` may be
        empty where no request has own tokens (one that has some gets a NaN row and sets status 512).  K/V have Q's dtype (no
        fp8), and a paged pool's pages lie one after another.  ``scale`` must be > 0.  The call can
        be captured (``DecodeGraph`` itself captures plain engines only).
        """
        if prefix.numel() * self.config.page_size > self.prefix_capacity:
            raise ValueError("prefix names more tokens than prefix_capacity")
        out = self.layers[layer]
        scale = self._default_scale if scale is None else float(scale)
        self._calls[layer] = (q, k, v, pages, indptr, out.output, out.partial, out.lse, out.counter, out.status,
                              self.plan.storage, self.plan.geometry, self.config.page_size, scale, float(logit_cap or 0.0),
                              1.0, 1.0, k_new, v_new, new_loc)
        self._decode_prefix(q, k, v, pages, indptr, out.output, out.partial, out.lse, out.counter, out.status,
                            self.plan.storage, self.plan.geometry, self.config.page_size, scale, float(logit_cap or 0.0),
                            k_new, v_new, new_loc, prefix, prefix_length, self.workspace)
        return out.output

    def kernel_kind(self, layer=0):
        """Name of the decode kernel of the own tokens ("none" for empty ``pages``); the small-batch kernel,
        which merges the splits itself, is never among them."""
        if self._calls[layer][3].numel() == 0:
            return "none"
        kind = super().kernel_kind(layer)
        return "mma.sync" if kind == "small" else kind
