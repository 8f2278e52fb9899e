//! Projections in 8-bit floating point and the norm before them (no file of the reference; next to its
//! RMSNorm, src/kernels/rmsnorm.zig:6-43, and QMatMulInt4, src/kernels/quantized.zig:6-51).  Every
//! forward() is synchronous; T is f32, f16 or u16 (the bits of a bf16).  Not built here (no Zig
//! toolchain on the build or GPU machines).
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

/// Blocks of 128 that n values make.
pub fn blocks(n: u32) u32 {
    return (n + 127) / 128;
}

/// Bytes from one row of k codes to the next that the product takes: on 16-byte boundaries.
pub fn rowOf(k: u32) u32 {
    return (k + 15) / 16 * 16;
}

/// Whether a buffer holds rows of dim elements, stride apart.
fn holds(count: usize, rows: u32, stride: u32, dim: u32) bool {
    return rows == 0 or count >= (@as(usize, rows) - 1) * stride + dim;
}

/// x + residual (null: x alone), its RMS norm as e4m3 codes [rows][dim] and scales
/// [rows][blocks(dim)], and the sum itself (a null sum_out: not written).  forward() takes as many
/// packed rows as codes hold, forwardRows() rows of codes that lie codes_stride bytes apart (0: dim;
/// LinearFP8 takes rowOf(k)).
pub const AddRMSNormFP8 = struct {
    device: *cuda.Device,

    pub fn init(device: *cuda.Device) !AddRMSNormFP8 {
        return .{ .device = device };
    }

    pub fn forward(
        self: *AddRMSNormFP8,
        comptime T: type,
        x: *cuda.Buffer(T),
        residual: ?*cuda.Buffer(T),
        weight: ?*cuda.Buffer(f32),
        sum_out: ?*cuda.Buffer(T),
        codes: *cuda.Buffer(u8),
        scales: *cuda.Buffer(f32),
        dim: u32,
        eps: f32,
    ) !void {
        try self.forwardRows(T, x, residual, weight, sum_out, codes, scales, dim, eps,
            @intCast(codes.count / dim), 0);
    }

    pub fn forwardRows(
        self: *AddRMSNormFP8,
        comptime T: type,
        x: *cuda.Buffer(T),
        residual: ?*cuda.Buffer(T),
        weight: ?*cuda.Buffer(f32),
        sum_out: ?*cuda.Buffer(T),
        codes: *cuda.Buffer(u8),
        scales: *cuda.Buffer(f32),
        dim: u32,
        eps: f32,
        rows: u32,
        codes_stride: u32,
    ) !void {
        const stride = if (codes_stride == 0) dim else codes_stride;
        if (!holds(x.count, rows, dim, dim) or !holds(codes.count, rows, stride, dim) or
            !holds(scales.count, rows, blocks(dim), blocks(dim))) return error.InvalidArgument;
        if (residual) |r| if (!holds(r.count, rows, dim, dim)) return error.InvalidArgument;
        if (sum_out) |t| if (!holds(t.count, rows, dim, dim)) return error.InvalidArgument;
        if (weight) |w| if (w.count < dim) return error.InvalidArgument;
        try cuda.check(c.tk_add_rmsnorm_fp8(self.device.ctx, x.handle,
            if (residual) |r| r.handle else null, if (weight) |w| w.handle else null,
            if (sum_out) |t| t.handle else null, codes.handle, scales.handle, rows, dim, 0, 0, 0,
            stride, eps, typeOf(T)));
    }
};

/// Codes and scales of activations that no norm precedes; forward() and forwardRows() as above.
pub const QuantizeFP8 = struct {
    device: *cuda.Device,

    pub fn init(device: *cuda.Device) !QuantizeFP8 {
        return .{ .device = device };
    }

    pub fn forward(
        self: *QuantizeFP8,
        comptime T: type,
        x: *cuda.Buffer(T),
        codes: *cuda.Buffer(u8),
        scales: *cuda.Buffer(f32),
        dim: u32,
    ) !void {
        try self.forwardRows(T, x, codes, scales, dim, @intCast(codes.count / dim), 0);
    }

    pub fn forwardRows(
        self: *QuantizeFP8,
        comptime T: type,
        x: *cuda.Buffer(T),
        codes: *cuda.Buffer(u8),
        scales: *cuda.Buffer(f32),
        dim: u32,
        rows: u32,
        codes_stride: u32,
    ) !void {
        const stride = if (codes_stride == 0) dim else codes_stride;
        if (!holds(x.count, rows, dim, dim) or !holds(codes.count, rows, stride, dim) or
            !holds(scales.count, rows, blocks(dim), blocks(dim))) return error.InvalidArgument;
        try cuda.check(c.tk_fp8_quantize(self.device.ctx, x.handle, codes.handle, scales.handle, rows,
            dim, 1, 0, stride, typeOf(T)));
    }
};

/// A weight [n][k] (out_dim, in_dim) in blocks of 128 x 128 that owns its buffers (rows of codes on
/// 16-byte boundaries), and the product with it.
pub const LinearFP8 = struct {
    device: *cuda.Device,
    n: u32,
    k: u32,
    row: u32,
    codes: cuda.Buffer(u8),
    scales: cuda.Buffer(f32),

    pub fn init(device: *cuda.Device, n: u32, k: u32) !LinearFP8 {
        const row = rowOf(k);
        var codes = try cuda.Buffer(u8).initKind(device, @as(usize, n) * row, c.TK_MEM_DEVICE);
        errdefer codes.deinit();
        return .{
            .device = device,
            .n = n,
            .k = k,
            .row = row,
            .codes = codes,
            .scales = try cuda.Buffer(f32).initKind(device, @as(usize, blocks(n)) * blocks(k), c.TK_MEM_DEVICE),
        };
    }

    pub fn deinit(self: *LinearFP8) void {
        self.codes.deinit();
        self.scales.deinit();
    }

    /// Quantises weight, n rows of k values.
    pub fn load(self: *LinearFP8, comptime T: type, weight: *cuda.Buffer(T)) !void {
        if (!holds(weight.count, self.n, self.k, self.k)) return error.InvalidArgument;
        try cuda.check(c.tk_fp8_quantize(self.device.ctx, weight.handle, self.codes.handle,
            self.scales.handle, self.n, self.k, 128, 0, self.row, typeOf(T)));
    }

    /// out [m][n] of m rows of activations, a_stride bytes apart (0: k).
    pub fn forward(
        self: *LinearFP8,
        comptime T: type,
        codes: *cuda.Buffer(u8),
        scales: *cuda.Buffer(f32),
        out: *cuda.Buffer(T),
        m: u32,
        a_stride: u32,
    ) !void {
        const stride = if (a_stride == 0) self.k else a_stride;
        if (!holds(codes.count, m, stride, self.k) or !holds(scales.count, m, blocks(self.k), blocks(self.k)) or
            !holds(out.count, m, self.n, self.n)) return error.InvalidArgument;
        try cuda.check(c.tk_fp8_matmul(self.device.ctx, codes.handle, scales.handle, self.codes.handle,
            self.scales.handle, out.handle, m, self.k, self.n, stride, self.row, 0, typeOf(T)));
    }
};
