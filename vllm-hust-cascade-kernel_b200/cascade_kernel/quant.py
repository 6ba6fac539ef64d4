"""A paged key-value cache held in 4 bits and the steps that serve from it.

``QuantCache`` keeps two pools per layer, keys and values, uint8
``[blocks, page, kv heads, 80]`` (the 80 bytes of a row: include/cascade_b200.h),
with the table, lengths and reference counts of ``LatentCache``, whose page
operators it shares. Rows are quantised as they are written
(``torch.ops.npu.cascade_quant_write``), read back into 16 or 32 bits
(``cascade_quant_read``) and attended to as they lie (``cascade_quant_decode``).
What the 4 bits cost shows in ``torch.ops.npu.cascade_token_logprobs`` of the
two models' logits.
"""
import torch

from .latent import LatentCache

DIM, GROUP, ROW = 128, 32, 80


class QuantCache(LatentCache):
    """Rows (sequences) over shared pages of 4-bit keys and values; rows, pages and errors as in ``LatentCache``.
    ``write`` and ``read`` wait for the device."""

    def __init__(self, layers, blocks, page, rows, cols, kv_heads, device="cuda"):
        self.page = page
        self.pools = [torch.zeros((blocks, page, kv_heads, ROW), dtype=torch.uint8, device=device) for _ in range(2 * layers)]
        self.table = torch.full((rows, cols), -1, dtype=torch.int32, device=device)
        self.lens = torch.zeros(rows, dtype=torch.int64, device=device)
        self.refs = torch.zeros(blocks, dtype=torch.int32, device=device)

    def slots(self, counts):
        """Slots of the last ``counts`` (host list) tokens of the rows, int64 [sum(counts)]: the same for every layer."""
        page, place = self._last(counts, "slots")
        return page * self.page + place

    def write(self, layer, key, value, slots):
        """Quantises ``key`` and ``value`` [tokens, kv heads, 128] into ``slots``, or into those of the last ``slots``
        (host list) tokens of the rows, which ``grow`` gave them."""
        torch.ops.npu.cascade_quant_write(key, value, *self.pools[2 * layer : 2 * layer + 2], self._slots(slots))

    def read(self, layer, slots, dtype=torch.bfloat16):
        """Keys and values [tokens, kv heads, 128] of ``slots``, or of the last ``slots`` (host list) tokens of the rows."""
        return torch.ops.npu.cascade_quant_read(*self.pools[2 * layer : 2 * layer + 2], self._slots(slots), dtype)

    def _slots(self, slots):
        return slots if isinstance(slots, torch.Tensor) else self.slots(slots)

    def attend(self, layer, query, q_len, scale, rows=None):
        """The last ``q_len`` tokens of every row (their queries [rows * q_len, heads, 128]) over the row's cache."""
        table, lens = (self.table, self.lens) if rows is None else (self.table[rows].contiguous(), self.lens[rows])
        return self._attend(layer, query, table, lens, q_len, scale, True)

    def attend_shared(self, layer, query, prefix_table, prefix_lens, scale, own_from):
        """One token per row whose first ``own_from`` tokens (whole pages; no row may be shorter) are one prefix shared by
        all rows: the prefix is one request of all rows' queries, each row's rest is read by itself, the two are merged."""
        if own_from % self.page:
            raise ValueError("attend_shared: the shared prefix must be whole pages")
        o1, l1 = self._attend(layer, query, prefix_table, prefix_lens, query.shape[0], scale, False)
        rest = self.table[:, own_from // self.page :].contiguous()
        o2, l2 = self._attend(layer, query, rest, self.lens - own_from, 1, scale, True)
        code = {torch.bfloat16: 1, torch.float16: 3}[query.dtype]
        return torch.ops.npu.cascade_lse_merge(o1, o2, l1, l2, code)

    def _attend(self, layer, query, table, lens, q_len, scale, causal):
        q_lens = torch.full_like(lens, q_len)
        return torch.ops.npu.cascade_quant_decode(query, *self.pools[2 * layer : 2 * layer + 2], table, q_lens, lens, q_len,
                                                  scale, causal)
