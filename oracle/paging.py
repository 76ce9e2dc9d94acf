"""Block tables and slot maps from request lengths, one request after the other in Python integers — test infrastructure
only. The rule is nanochat_amd/paging.py's: pages in slot order while the pool has enough, then rows in slot order while
the step has enough, all or nothing a slot; the free list is a stack.

Pinned by tests/test_oracle_paging.py: no page is held twice or lost, refusals begin where the pages or rows end, and a
trim to the old lengths undoes an extend."""
PAGE = 16


def pages_of(length):
    return -(-length // PAGE)


class BlockTables:
    """Lists in place of the device tensors of the same names; free holds the free pages, the next one last."""

    def __init__(self, slots, max_pages, num_pages):
        self.table = [[-1] * max_pages for _ in range(slots)]
        self.lengths = [0] * slots
        self.free = list(range(num_pages - 1, -1, -1))

    def extend(self, new_tokens, rows):
        """-> (cu_seqlens, positions, slot_map, granted)."""
        cap = len(self.table[0]) * PAGE
        asked = [max(n, 0) if length + max(n, 0) <= cap else 0 for n, length in zip(new_tokens, self.lengths)]
        need = [pages_of(length + n) - pages_of(length) for n, length in zip(asked, self.lengths)]
        out_of_pages = False
        for b, k in enumerate(need):
            out_of_pages = out_of_pages or sum(need[:b + 1]) > len(self.free)
            if k and out_of_pages:
                asked[b] = 0
        cu, positions, slot_map, granted = [0], [], [], []
        wanted = 0
        for b, n in enumerate(asked):
            wanted += n
            granted.append(n if wanted <= rows else 0)
            for p in range(self.lengths[b], self.lengths[b] + granted[b]):
                if p % PAGE == 0:
                    self.table[b][p // PAGE] = self.free.pop()
                positions.append(p)
                slot_map.append(self.table[b][p // PAGE] * PAGE + p % PAGE)
            self.lengths[b] += granted[b]
            cu.append(len(positions))
        pad = [-1] * (rows - len(positions))
        return cu, positions + pad, slot_map + pad, granted

    def trim(self, keep):
        freed = []
        for b, n in enumerate(keep):
            if 0 <= n < self.lengths[b]:
                for p in range(pages_of(n), pages_of(self.lengths[b])):
                    freed.append(self.table[b][p])
                    self.table[b][p] = -1
                self.lengths[b] = n
        self.free += freed[::-1]
