"""A paged latent cache and the steps that serve from it.

``LatentCache`` keeps what the page operators read and write: one pool per
layer ``[blocks, page, 576]`` (512 latent values and 64 rotary key values per
token), a block table, the rows' lengths and the pages' reference counts. The
operators return the new table, lengths and counts; the cache swaps them in.
Attention over it is ``torch.ops.npu.cascade_latent_decode`` (absorbed form);
prompts attend in the expanded form, ``torch.ops.npu.cascade_latent_prefill``,
and drafted tokens are checked by ``torch.ops.npu.cascade_verify_drafts``.
"""
import torch

LATENT, ROPE = 512, 64


class LatentCache:
    """Rows (sequences) over shared pages. A row of length -1 could not be made: it stays so, neither grows nor forks, until
    it is cut to 0 tokens. ``grow`` and ``write`` wait for the device (what they cannot do raises), the others do not."""

    def __init__(self, layers, blocks, page, rows, cols, dtype=torch.bfloat16, device="cuda"):
        self.page = page
        self.pools = [torch.zeros((blocks, page, LATENT + ROPE), dtype=dtype, device=device) for _ in range(layers)]
        self.table = torch.full((rows, cols), -1, dtype=torch.int32, device=device)
        self.lens = torch.zeros(rows, dtype=torch.int64, device=device)
        self.refs = torch.zeros(blocks, dtype=torch.int32, device=device)

    def grow(self, tokens):
        """Gives every row the pages for ``tokens`` (int64 [rows]) more tokens, free ones in ascending order, and
        lengthens it. A row that goes on inside a page that others hold too (``truncate`` cut it there) gets a copy of
        the page first; if all its holders go on, the lowest row keeps it. Raises, and changes nothing, if the pages or
        the table's columns run out, and for a row that cannot grow."""
        cols, page = self.table.shape[1], self.page
        grown = self.lens + tokens
        have, want = (self.lens + page - 1) // page, (grown + page - 1) // page
        free = torch.nonzero(self.refs == 0).squeeze(1)
        # one look at the host: pages needed, rows inside a shared page, rows past the columns, rows that cannot grow
        inside = (self.lens % page > 0) & (tokens > 0)
        end = self.lens.clamp(0, max(cols * page - 1, 0)) // page
        old = self.table.gather(1, end[:, None]).squeeze(1).long() if cols else torch.zeros_like(end)
        shared = inside & (self.refs[old] > 1) if free.numel() < self.refs.numel() else torch.zeros_like(inside)
        bad = (tokens < 0) | ((self.lens < 0) & (tokens > 0))
        need, some, over, wrong = torch.stack((want - have, shared, want > cols, bad)).sum(1).tolist()
        if wrong:
            raise RuntimeError(f"LatentCache.grow: row {int(torch.nonzero(bad)[0])} could not be made (length -1), or its "
                               "tokens are negative")
        row = self._leaving(shared, inside, old) if some else end[:0]
        total = need + row.numel()
        if total > free.numel() or over:
            raise RuntimeError(f"LatentCache: {total} pages needed, {free.numel()} free, {cols} columns")
        if row.numel():
            copies = free[need:total]
            torch.ops.npu.cascade_page_copy(self.pools, old[row], copies)
            self.refs.index_add_(0, old[row], torch.full_like(self.refs[copies], -1))
            self.table[row, end[row]] = copies.int()
        if total:
            col = torch.arange(cols, device=end.device)
            self.table.masked_scatter_((col >= have[:, None]) & (col < want[:, None]), free[:total].int())
            self.refs.index_fill_(0, free[:total], 1)
        self.lens = grown

    def _leaving(self, shared, inside, page):
        """The rows of `shared` that have to leave their last page `page` to others: all but the lowest one if every holder
        goes on inside it."""
        row, rows = torch.nonzero(inside).squeeze(1), inside.numel()
        at = page[row]
        going = torch.bincount(at, minlength=self.refs.numel())
        first = torch.full_like(going, rows).scatter_reduce_(0, at, row, "amin")
        return row[shared[row] & ((going[at] < self.refs[at]) | (first[at] < row))]

    def write(self, layer, latents, counts):
        """Stores ``latents`` [sum(counts), 576] as the last ``counts`` (host list) tokens of the rows, which ``grow`` gave
        them."""
        if len(counts) > self.table.shape[0]:
            raise RuntimeError(f"LatentCache.write: {len(counts)} counts, {self.table.shape[0]} rows")
        rows = torch.repeat_interleave(torch.arange(len(counts)), torch.tensor(counts))
        rows, back = torch.stack((rows, torch.cat([torch.arange(n, 0, -1) for n in counts]))).to(self.table.device)
        at = self.lens[rows] - back
        if bool((at < 0).any()):
            raise RuntimeError(f"LatentCache.write: row {int(rows[at < 0][0])} has no token there")
        page = self.table[rows, at // self.page].long()
        self.pools[layer][page, at % self.page] = latents

    def attend(self, layer, query, q_len, scale, rows=None):
        """The last ``q_len`` tokens of every row (their queries [rows * q_len, heads, 576]) over the row's cache."""
        table, lens = (self.table, self.lens) if rows is None else (self.table[rows].contiguous(), self.lens[rows])
        ones = torch.full_like(lens, q_len)
        return torch.ops.npu.cascade_latent_decode(query, self.pools[layer], table, ones, lens, q_len, scale, True)

    def attend_shared(self, layer, query, prefix_table, prefix_lens, scale, own_from):
        """One token per row whose first ``own_from`` tokens (whole pages; no row may be shorter) are one prefix shared by
        all rows. The prefix is one request of all rows' queries, read once per 128 of its [row x head] query rows (per
        16 or 32 if there are no more), not once per row; each row's rest is read by itself, and the two are merged."""
        B = query.shape[0]
        skip = own_from // self.page
        if own_from % self.page:
            raise ValueError("attend_shared: the shared prefix must be whole pages")
        qs = torch.full_like(prefix_lens, B)
        o1, l1 = torch.ops.npu.cascade_latent_decode(query, self.pools[layer], prefix_table, qs, prefix_lens, B, scale, False)
        rest = self.table[:, skip:].contiguous()
        ones = torch.ones_like(self.lens)
        o2, l2 = torch.ops.npu.cascade_latent_decode(query, self.pools[layer], rest, ones, self.lens - own_from, 1, scale, True)
        code = {torch.bfloat16: 1, torch.float16: 3}[query.dtype]
        return torch.ops.npu.cascade_lse_merge(o1, o2, l1, l2, code)

    def fork(self, parents):
        """The rows become copies of rows ``parents`` (int64): shared full pages, an own copy of a partly filled last
        one. The old rows give their pages back afterwards, so the copies need free pages: a row that found none, or
        whose parent could not be made, has length -1 (attention over it sees nothing)."""
        child, lens, refs = torch.ops.npu.cascade_page_fork(self.pools, self.table, self.lens, self.refs, parents)
        _, _, refs = torch.ops.npu.cascade_page_free(self.table, self.lens, refs, torch.zeros_like(self.lens), self.page)
        self.table, self.lens, self.refs = child, lens, refs

    def truncate(self, keep):
        """Cuts the rows to ``keep`` tokens (int64 [rows]) and frees the pages past them. 0 empties a row, one that could
        not be made as well."""
        made = (self.lens >= 0) | (keep <= 0)
        self.table, lens, self.refs = torch.ops.npu.cascade_page_free(self.table, self.lens, self.refs, keep, self.page)
        self.lens = torch.where(made, lens, -1)

    def compact(self):
        """Moves the live pages to the front of the pools; returns their number (int32 [1], on the device)."""
        self.table, self.refs, live = torch.ops.npu.cascade_page_compact(self.pools, self.table, self.lens, self.refs)
        return live
