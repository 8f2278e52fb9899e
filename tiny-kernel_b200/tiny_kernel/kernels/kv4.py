"""The serving step over a key/value cache held in 4 bits (no file of the reference; next to its
PagedAttention, src/kernels/attention.zig:51-100).  Every forward() is synchronous; streams and
graphs go through the functions of ops."""
from __future__ import annotations

from .. import _lib, ops


class PagedSlots:
    """Block tables, positions and slots of a step from the requests' lengths (i32 buffers)."""

    def __init__(self, device):
        self.device = device

    @classmethod
    def init(cls, device) -> "PagedSlots":
        return cls(device)

    def forward(self, context_lens, query_lens, free_blocks, free_range, block_tables, kv_lens,
                query_start, positions, slots, counts, block_size, num_blocks):
        batch = context_lens.count
        ops.paged_slots(self.device, context_lens, query_lens, free_blocks, free_range,
                        block_tables, kv_lens, query_start, positions, slots, counts, batch,
                        block_tables.count // batch, block_size, num_blocks, slots.count)


class QKNormRoPE:
    """Norm of each head of queries and keys (a None weight: none) and their rotation."""

    def __init__(self, device):
        self.device = device

    @classmethod
    def init(cls, device) -> "QKNormRoPE":
        return cls(device)

    def forward(self, q, k, q_weight, k_weight, cos_cache, sin_cache, positions, q_out, k_out,
                q_heads, kv_heads, head_dim, rot_dim, max_pos, eps, dtype="f32",
                interleaved=False):
        ops.qk_norm_rope(self.device, q, k, q_weight, k_weight, cos_cache, sin_cache, positions,
                         q_out, k_out, positions.count, q_heads, kv_heads, head_dim, rot_dim,
                         max_pos, eps, dtype, interleaved)


class KV4Cache:
    """A cache of num_blocks pages that owns its buffers (device memory), and the calls on it.  The
    workspace of forward() is the object's: one forward() at a time."""

    def __init__(self, device, num_blocks, kv_heads, block_size, head_dim, group_size):
        self.device = device
        rows = num_blocks * kv_heads * block_size
        alloc = lambda dtype, count: device.create_buffer(dtype, count, _lib.TK_MEM_DEVICE)
        self.k_codes, self.v_codes = (alloc("u8", rows * (head_dim // 2)) for _ in "kv")
        self.k_scales, self.v_scales = (alloc("u16", rows * (head_dim // group_size) * 2)
                                        for _ in "kv")
        self.cache = ops.kv4_cache(self.k_codes, self.v_codes, self.k_scales, self.v_scales,
                                   num_blocks, kv_heads, block_size, head_dim, group_size)
        self.workspace = None

    @classmethod
    def init(cls, device, num_blocks, kv_heads, block_size, head_dim, group_size) -> "KV4Cache":
        return cls(device, num_blocks, kv_heads, block_size, head_dim, group_size)

    def append(self, k, v, slots, dtype="f32"):
        ops.kv4_append(self.device, self.cache, k, v, slots, slots.count, dtype)

    def gather(self, slots, k, v, dtype="f32"):
        ops.kv4_gather(self.device, self.cache, slots, k, v, slots.count, dtype)

    def forward(self, q, block_tables, kv_lens, query_start, o, q_heads, scale, dtype="f32"):
        """o = attention of the step's queries (query_start None: one token per sequence)."""
        size = ops.kv4_attention_workspace(self.device, self.cache, q_heads)
        if self.workspace is None or self.workspace.count < size:
            self.workspace = self.device.create_buffer("u8", size, _lib.TK_MEM_DEVICE)
        batch = kv_lens.count
        ops.kv4_attention(self.device, self.cache, q, block_tables, kv_lens, query_start, o,
                          self.workspace, size, q.count // (q_heads * self.cache.head_dim), batch,
                          q_heads, block_tables.count // batch, scale, dtype)

    def deinit(self) -> None:
        for b in (self.k_codes, self.v_codes, self.k_scales, self.v_scales, self.workspace):
            if b is not None:
                b.deinit()
        self.workspace = None
