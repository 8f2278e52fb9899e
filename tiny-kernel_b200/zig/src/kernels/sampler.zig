//! The choice of tokens for a batch (next to the reference's softmax_sample,
//! src/kernels/shaders.zig:826-887).  Synchronous; T is f32, f16 or u16 (the bits of a bf16).  Not
//! built here (no Zig toolchain on the build or GPU machines).
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

/// tokens[row] of each row of logits by its temperature, top_k, top_p and min_p, each a buffer of rows
/// or null, and its random number in [0, 1); kept[row] (or null) = tokens that the filters leave.
pub const SampleTokens = struct {
    device: *cuda.Device,

    pub fn init(device: *cuda.Device) !SampleTokens {
        return .{ .device = device };
    }

    pub fn forward(
        self: *SampleTokens,
        comptime T: type,
        logits: *cuda.Buffer(T),
        temperature: ?*cuda.Buffer(f32),
        top_k: ?*cuda.Buffer(i32),
        top_p: ?*cuda.Buffer(f32),
        min_p: ?*cuda.Buffer(f32),
        random: *cuda.Buffer(f32),
        tokens: *cuda.Buffer(i32),
        kept: ?*cuda.Buffer(i32),
    ) !void {
        const rows: u32 = @intCast(tokens.count);
        const vocab: u32 = @intCast(logits.count / tokens.count);
        try cuda.check(c.tk_sample_tokens(self.device.ctx, logits.handle,
            if (temperature) |t| t.handle else null, if (top_k) |t| t.handle else null,
            if (top_p) |t| t.handle else null, if (min_p) |t| t.handle else null, random.handle,
            tokens.handle, if (kept) |t| t.handle else null, rows, vocab, 0, typeOf(T)));
    }
};
