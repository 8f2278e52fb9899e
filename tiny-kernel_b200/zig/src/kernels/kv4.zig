//! The serving step over a key/value cache held in 4 bits (no file of the reference; next to its
//! PagedAttention, src/kernels/attention.zig:51-100).  Every forward() is synchronous; T is f32,
//! f16 or u16 (the bits of a bf16).  Not built here (no Zig toolchain on the build or GPU machines).
const cuda = @import("../cuda/cuda.zig");
const c = cuda.c;

fn typeOf(comptime T: type) c_int {
    return switch (T) {
        f32 => c.TK_F32,
        f16 => c.TK_F16,
        u16 => c.TK_BF16,
        else => @compileError("f32, f16 or u16 (bf16)"),
    };
}

/// Block tables, positions and slots of a step from the requests' lengths.
pub const PagedSlots = struct {
    device: *cuda.Device,

    pub fn init(device: *cuda.Device) !PagedSlots {
        return .{ .device = device };
    }

    pub fn forward(
        self: *PagedSlots,
        context_lens: *cuda.Buffer(i32),
        query_lens: *cuda.Buffer(i32),
        free_blocks: *cuda.Buffer(i32),
        free_range: *cuda.Buffer(i32),
        block_tables: *cuda.Buffer(i32),
        kv_lens: *cuda.Buffer(i32),
        query_start: *cuda.Buffer(i32),
        positions: *cuda.Buffer(i32),
        slots: *cuda.Buffer(i32),
        counts: *cuda.Buffer(i32),
        block_size: u32,
        num_blocks: u32,
    ) !void {
        const batch: u32 = @intCast(context_lens.count);
        const max_blocks: u32 = @intCast(block_tables.count / batch);
        const max_tokens: u32 = @intCast(slots.count);
        try cuda.check(c.tk_paged_slots(self.device.ctx, context_lens.handle, query_lens.handle,
            free_blocks.handle, free_range.handle, block_tables.handle, kv_lens.handle,
            query_start.handle, positions.handle, slots.handle, counts.handle, batch, max_blocks,
            block_size, num_blocks, max_tokens));
    }
};

/// Norm of each head of queries and keys (a null weight: none) and their rotation.
pub const QKNormRoPE = struct {
    device: *cuda.Device,

    pub fn init(device: *cuda.Device) !QKNormRoPE {
        return .{ .device = device };
    }

    pub fn forward(
        self: *QKNormRoPE,
        comptime T: type,
        q: *cuda.Buffer(T),
        k: *cuda.Buffer(T),
        q_weight: ?*cuda.Buffer(f32),
        k_weight: ?*cuda.Buffer(f32),
        cos_cache: *cuda.Buffer(f32),
        sin_cache: *cuda.Buffer(f32),
        positions: *cuda.Buffer(i32),
        q_out: *cuda.Buffer(T),
        k_out: *cuda.Buffer(T),
        q_heads: u32,
        kv_heads: u32,
        head_dim: u32,
        rot_dim: u32,
        max_pos: u32,
        eps: f32,
        interleaved: bool,
    ) !void {
        const tokens: u32 = @intCast(positions.count);
        const flags: u32 = if (interleaved) c.TK_ROPE_INTERLEAVED else 0;
        try cuda.check(c.tk_qk_norm_rope(self.device.ctx, q.handle, k.handle,
            if (q_weight) |w| w.handle else null, if (k_weight) |w| w.handle else null,
            cos_cache.handle, sin_cache.handle, positions.handle, q_out.handle, k_out.handle, tokens,
            q_heads, kv_heads, head_dim, rot_dim, max_pos, 0, 0, 0, 0, eps, typeOf(T), flags));
    }
};

/// A cache of num_blocks pages that owns its buffers, and the calls on it; one forward() at a time
/// (the workspace is the cache's).
pub const KV4Cache = struct {
    device: *cuda.Device,
    k_codes: cuda.Buffer(u8),
    v_codes: cuda.Buffer(u8),
    k_scales: cuda.Buffer(u16),
    v_scales: cuda.Buffer(u16),
    workspace: ?cuda.Buffer(u8),
    cache: c.tk_kv4_cache,

    pub fn init(
        device: *cuda.Device,
        num_blocks: u32,
        kv_heads: u32,
        block_size: u32,
        head_dim: u32,
        group_size: u32,
    ) !KV4Cache {
        const rows: usize = @as(usize, num_blocks) * kv_heads * block_size;
        const codes = rows * (head_dim / 2);
        const pairs = rows * (head_dim / group_size) * 2;
        const kind = c.TK_MEM_DEVICE;
        var k_codes = try cuda.Buffer(u8).initKind(device, codes, kind);
        errdefer k_codes.deinit();
        var v_codes = try cuda.Buffer(u8).initKind(device, codes, kind);
        errdefer v_codes.deinit();
        var k_scales = try cuda.Buffer(u16).initKind(device, pairs, kind);
        errdefer k_scales.deinit();
        const v_scales = try cuda.Buffer(u16).initKind(device, pairs, kind);
        return .{
            .device = device,
            .k_codes = k_codes,
            .v_codes = v_codes,
            .k_scales = k_scales,
            .v_scales = v_scales,
            .workspace = null,
            .cache = .{
                .k_codes = k_codes.handle,
                .v_codes = v_codes.handle,
                .k_scales = k_scales.handle,
                .v_scales = v_scales.handle,
                .num_blocks = num_blocks,
                .kv_heads = kv_heads,
                .block_size = block_size,
                .head_dim = head_dim,
                .group_size = group_size,
            },
        };
    }

    pub fn deinit(self: *KV4Cache) void {
        self.k_codes.deinit();
        self.v_codes.deinit();
        self.k_scales.deinit();
        self.v_scales.deinit();
        if (self.workspace) |*w| w.deinit();
    }

    pub fn append(self: *KV4Cache, comptime T: type, k: *cuda.Buffer(T), v: *cuda.Buffer(T),
        slots: *cuda.Buffer(i32)) !void {
        const tokens: u32 = @intCast(slots.count);
        try cuda.check(c.tk_kv4_append(self.device.ctx, &self.cache, k.handle, v.handle, slots.handle,
            tokens, 0, 0, typeOf(T)));
    }

    pub fn gather(self: *KV4Cache, comptime T: type, slots: *cuda.Buffer(i32), k: *cuda.Buffer(T),
        v: *cuda.Buffer(T)) !void {
        const tokens: u32 = @intCast(slots.count);
        try cuda.check(c.tk_kv4_gather(self.device.ctx, &self.cache, slots.handle, k.handle, v.handle,
            tokens, 0, 0, typeOf(T)));
    }

    /// query_start null: one token per sequence.
    pub fn forward(
        self: *KV4Cache,
        comptime T: type,
        q: *cuda.Buffer(T),
        block_tables: *cuda.Buffer(i32),
        kv_lens: *cuda.Buffer(i32),
        query_start: ?*cuda.Buffer(i32),
        o: *cuda.Buffer(T),
        q_heads: u32,
        scale: f32,
    ) !void {
        var need: usize = 0;
        try cuda.check(c.tk_kv4_attention_workspace(self.device.ctx, &self.cache, q_heads, &need));
        if (self.workspace == null)
            self.workspace = try cuda.Buffer(u8).initKind(self.device, need, c.TK_MEM_DEVICE);
        const batch: u32 = @intCast(kv_lens.count);
        const tokens: u32 = @intCast(q.count / (@as(usize, q_heads) * self.cache.head_dim));
        const max_blocks: u32 = @intCast(block_tables.count / batch);
        try cuda.check(c.tk_kv4_attention(self.device.ctx, &self.cache, q.handle, block_tables.handle,
            kv_lens.handle, if (query_start) |s| s.handle else null, o.handle, self.workspace.?.handle,
            self.workspace.?.count, tokens, batch, q_heads, max_blocks, 0, 0, scale, typeOf(T)));
    }
};
