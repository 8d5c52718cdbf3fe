"""K/V cache held in 4 or 8 bits: rows quantised as they are written, read back, and attended to.

64 consecutive dims of one token and head are a group.  With N = 15 (4 bits) or 255 (8 bits) a
group is held as whole numbers n in 0..N, a scale s and an offset z in bf16: z is the group's
minimum rounded down, s is (maximum - z) / N rounded up, n is (x - z) / s rounded to the nearest
(ties to even; 0 where s is 0), and the value held is s n + z.  That is 4.5 or 8.5 bits a value.  A group with a
NaN, an infinity or a magnitude above 2^126 reads back as NaN.

The attention is that of the values held, in 32 bits, and its output's own rounding decides its error, with two
exceptions for bf16 queries: weights are rounded to f16 (2^-11), and in steps with many query slots of a sequence
(rows x q heads of a kv head: more than 32, or 16 with 256 dims) K and V are too, down to 2^-16 (V of 4 bits: 2^-20)
of their token's largest scale.  What a row does not see changes none of its bits.  Scores may have any size that 32
bits hold; K or V below 2^-64 in magnitude lose precision.

A ``QuantCache`` is the paged cache of a model's attention layers; a ``QuantAttention`` plans a
step's attention over it (``update``, once a step) and runs it (``attend``, once a layer).  All
calls run on the current stream with no host round trip, so a step can be captured in a CUDA
graph.  What only the device can see (a slot or page outside the cache, sequence boundaries
that do not fit) sets an error word that ``check()`` reads.
"""

from __future__ import annotations

import torch

from . import _ext

GROUP = 64    # dims that share a scale and an offset
BLOCK = 16    # tokens that are stored together
HEAD_DIMS = (64, 128, 256)
PAGE_SIZES = (16, 32, 64, 128, 256)


class QuantCache:
    """``data``: uint8 [layers, pages, bytes of a page], which a ``PagePool`` takes as one of its caches.
    Page-table rows name a sequence's pages in order, as for the bf16 caches."""

    def __init__(self, layers: int, num_pages: int, num_kv_heads: int, head_dim: int, bits: int = 4, page_size: int = 16,
                 device="cuda"):
        if bits not in (4, 8):
            raise ValueError(f"bits must be 4 or 8, got {bits}")
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {head_dim}")
        if page_size not in PAGE_SIZES:
            raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {page_size}")
        if layers < 1 or num_pages < 1 or num_kv_heads < 1:
            raise ValueError("layers, num_pages and num_kv_heads must be positive")
        C = _ext.load()
        self.layers, self.num_pages, self.num_kv_heads = layers, num_pages, num_kv_heads
        self.head_dim, self.bits, self.page_size = head_dim, bits, page_size
        self.page_bytes = num_kv_heads * (page_size // BLOCK) * C.quant_block_bytes(head_dim, bits)
        self.data = torch.zeros(layers, num_pages, self.page_bytes, dtype=torch.uint8, device=device)
        self.err = torch.zeros(1, dtype=torch.int32, device=device)
        self.state = C.QuantCacheState(self.data, num_kv_heads, head_dim, bits, page_size, self.err)

    def write(self, layer: int, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor, slots: torch.Tensor,
              positions: torch.Tensor) -> None:
        """Quantise the rows ``k`` and ``v`` [rows, kv heads, dim] (bf16 or f16; rows and heads may be strided)
        into token ``positions`` [rows] (int32) of the sequences ``slots`` [rows] (int32; rows of ``page_table``).
        A row with a negative position is not written.  Two rows must not name one place."""
        self.state.write(layer, k, v, page_table, slots, positions)

    def read(self, layer: int, page_table: torch.Tensor, slots: torch.Tensor, positions: torch.Tensor,
             dtype: torch.dtype = torch.bfloat16, k: torch.Tensor | None = None,
             v: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """The values held at ``positions`` of ``slots``: two tensors [rows, kv heads, dim] of ``dtype`` (bf16, f16 or
        f32), or ``k`` and ``v`` (of one such type; rows and heads may be strided) where they are given.  A row with
        a negative position is 0."""
        return self.state.read(layer, page_table, slots, positions, dtype, k, v)

    def check(self) -> None:
        """Raise if a write or read since the last check named a place outside the cache (reads the error word)."""
        if int(self.err.item()):
            self.err.zero_()
            raise RuntimeError("quantised cache: a slot, position or page outside the cache")


class QuantAttention:
    """Grouped-query attention of a step's rows over a ``QuantCache``.

    ``max_rows`` rows of ``max_seqs`` sequences at most (as many as rows unless given), ``max_seq_rows`` of one
    sequence: 1 for decode steps, the drafts + 1 of a verify step, the longest chunk of a prefill step.  Its
    workspace holds one step: calls of one object follow one another on a stream."""

    def __init__(self, cache: QuantCache, num_q_heads: int, max_rows: int, max_seqs: int | None = None, max_seq_rows: int = 1):
        self.cache, self.num_q_heads = cache, num_q_heads
        self.max_rows, self.max_seqs, self.max_seq_rows = max_rows, max_rows if max_seqs is None else max_seqs, max_seq_rows
        self.err = torch.zeros(1, dtype=torch.int32, device=cache.data.device)
        self.state = _ext.load().QuantPlanState(cache.state, num_q_heads, max_rows, self.max_seqs, max_seq_rows, self.err)

    def update(self, slots: torch.Tensor, seq_lens: torch.Tensor, seq_start: torch.Tensor | None = None) -> None:
        """Divide a step's keys over the GPU.  ``slots`` [rows] and ``seq_lens`` [rows] (int32): the sequence of each
        row and the keys it sees (0: none).  ``seq_start`` [sequences + 1] (int32): rows seq_start[i] to
        seq_start[i+1] are of one sequence (the first row's slot) and read its keys together; None: every row reads
        its own."""
        self.state.update(slots, seq_lens, seq_start)

    def attend(self, layer: int, q: torch.Tensor, page_table: torch.Tensor, sm_scale: float, gate: torch.Tensor | None = None,
               out: torch.Tensor | None = None, out_q: torch.Tensor | None = None,
               out_sf: torch.Tensor | None = None) -> torch.Tensor | None:
        """sigmoid(gate) * attention of ``q`` [rows, q heads, dim] (bf16 or f16; rows and heads may be strided) for
        the rows of the last ``update``; ``gate`` None: no gate.  The result goes to ``out`` ([rows, heads * dim]
        of q's type, allocated unless the MXFP8 pair ``out_q``, ``out_sf`` is given alone).  A row without keys, or
        of no sequence, gives 0; a head of ``q`` with a NaN or a magnitude of 2^101 or more gives NaN."""
        return self.state.attend(self.cache.state, layer, q, page_table, sm_scale, gate, out, out_q, out_sf)

    def check(self) -> None:
        """Raise if a call since the last check met a slot, page or sequence that does not fit (reads the error word)."""
        code = int(self.err.item())
        if code:
            self.err.zero_()
            raise RuntimeError(f"quantised attention: kernel error status {code}")
