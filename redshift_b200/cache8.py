"""An attention layer's K/V cache in 8 bits, as a decode loop keeps it.

``Cache8`` owns the buffers of ``qv_attention8`` for one layer (2,048.5 bytes a position instead of
4,096, and a tail of fp16 rows) and packs the tail's oldest block whenever it is complete::

    cache = Cache8(hot, context=32768)
    cache.load(key_rows, value_rows, n)            # after an fp16 prefill of n tokens, if any
    cache.attention(out, q_gate, key, value, q_norm, k_norm, batch, position)

``position`` is the caller's count of kept tokens: after a verify of 8 tokens of which 3 were kept
the next call simply passes a position that is 3 higher.  Rows from ``position`` on are never
packed, so nothing has to be rolled back.  The host keeps count of the rows and of what is packed, so
``attention``, ``pack`` and ``load`` are refused under graph capture: a replay would write the tail rows
of one position again, which hold others once the ring has gone on.  Capture ``HotPath.attention8``
itself where one position is to be replayed.
"""
BLOCK = 64


class Cache8:
    def __init__(self, hot, context, device='cuda', tail_rows=128):
        import torch
        if context < 1 or context > 139264:
            raise ValueError('context must be between 1 and 139264')
        if tail_rows % BLOCK or tail_rows < 2 * BLOCK:
            raise ValueError('the tail holds whole blocks of 64 rows, two or more')
        self.hot, self.context = hot, context
        dev = torch.device(device)
        if dev.index is None:
            dev = torch.device(dev.type, torch.cuda.current_device())
        blocks = -(-context // BLOCK)
        self.key_codes = torch.zeros((blocks, 4, BLOCK, 256), dtype=torch.int8, device=dev)
        self.value_codes = torch.zeros_like(self.key_codes)
        self.key_scales = torch.zeros((blocks, 4), device=dev)
        self.value_scales = torch.zeros_like(self.key_scales)
        self.key_tail = torch.zeros((tail_rows, 4, 256), dtype=torch.float16, device=dev)
        self.value_tail = torch.zeros_like(self.key_tail)
        self.packed = 0                  # positions in the packed part
        self.rows = 0                    # positions that hold a row

    def _not_captured(self):
        if self.hot.capturing(self.key_codes.device):
            raise RuntimeError('the cache cannot be changed under graph capture: a replay would write rows that have gone on')

    def _packed_buffers(self):
        return self.key_codes, self.key_scales, self.value_codes, self.value_scales

    def pack(self, position):
        """Pack the blocks that are complete before `position`, a number of kept tokens."""
        if not 0 <= position <= self.rows:
            raise ValueError(f'position {position} cannot be packed: the cache holds {self.rows} rows')
        end = position // BLOCK * BLOCK
        if end > self.packed:
            self._not_captured()
            self.hot.cache8_pack(*self._packed_buffers(), self.key_tail, self.value_tail, self.packed, end)
            self.packed = end

    def load(self, key_rows, value_rows, rows):
        """Take over the first `rows` positions of an fp16 cache [>= rows][4][256]: whole blocks packed,
        the rest into the tail."""
        if not 0 <= rows <= min(self.context, key_rows.shape[0], value_rows.shape[0]):
            raise ValueError('rows exceed the context or the given cache')
        self._not_captured()
        if rows == 0:
            self.packed = self.rows = 0
            return
        end = rows // BLOCK * BLOCK
        key_rows, value_rows = key_rows[:rows], value_rows[:rows]
        self.hot.cache8_pack(*self._packed_buffers(), key_rows, value_rows, 0, end)
        if rows > end:
            at = end % self.key_tail.shape[0]        # whole blocks: the rest does not wrap
            self.key_tail[at:at + rows - end].copy_(key_rows[end:rows])
            self.value_tail[at:at + rows - end].copy_(value_rows[end:rows])
        self.packed, self.rows = end, rows

    def unload(self, key_rows, value_rows, position):
        """Write the first `position` positions as fp16 rows, e.g. to prefill a further block behind them."""
        if not self.packed <= position <= min(self.rows, key_rows.shape[0], value_rows.shape[0]):
            raise ValueError('position is outside the cache or the given rows')
        if position == 0:
            return
        import torch
        key_rows, value_rows = key_rows[:position], value_rows[:position]
        self.hot.cache8_unpack(key_rows, value_rows, *self._packed_buffers(), 0, self.packed)
        tail = torch.arange(self.packed, position, device=self.key_tail.device) % self.key_tail.shape[0]
        key_rows[self.packed:] = self.key_tail[tail]
        value_rows[self.packed:] = self.value_tail[tail]

    def attention(self, out, q_gate, key, value, q_norm, k_norm, batch, position, epsilon=1e-6, workspace=None):
        """qv_attention8 for `batch` new tokens at `position`, after packing what is complete before it."""
        if position < self.packed:
            raise ValueError(f'position {position} lies in the packed part (up to {self.packed})')
        if position + batch > self.context:
            raise ValueError(f'the cache holds {self.context} positions')
        if position > self.rows:
            raise ValueError(f'position {position} leaves a gap: the cache holds {self.rows} rows')
        self._not_captured()
        self.pack(position)
        self.hot.attention8(out, *self._packed_buffers(), self.packed, self.key_tail, self.value_tail, q_gate, key,
                            value, q_norm, k_norm, batch, position, epsilon, workspace)
        self.rows = position + batch
