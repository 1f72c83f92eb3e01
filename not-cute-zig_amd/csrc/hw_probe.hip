// hw_probe.hip — single-wave probes of the gfx950 instruction semantics flash_fwd.hip and paged4.hip are built on.
//
// Not part of the flash path: the GPU tests load this code object and compare each probe's output
// with the layout the kernels assume, so a change of hardware or compiler behaviour shows up as a
// named failure instead of a parity mismatch somewhere in a kernel. Each kernel is launched with
// one workgroup of 64 threads and touches only the buffers the test sizes for it.
//
//   nc_probe_mfma32x32x16   v_mfma_f32_32x32x16_{f16,bf16}: operand and accumulator lane layout
//   nc_probe_ds_read_tr     ds_read_b64_tr_b16: which LDS elements each lane of a 16-lane group gets
//   nc_probe_permlane32     v_permlane32_swap: the lane-pair exchange used for row max / row sum
//   nc_probe_mfma_fp4_fp8   v_mfma_scale_f32_16x16x128_f8f6f4, 4-bit rows times 8-bit columns: lane layout and scales
//   nc_probe_mfma_fp4_fp6   the same with 6-bit columns
//   nc_probe_fp4_convert, nc_probe_fp8_convert, nc_probe_fp8_scaled, nc_probe_fp6_convert   rounding and order of the conversions to
//                           and from 4, 8 and 6 bits

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));

}  // namespace

// a: 32x16 row-major (A), b: 16x32 row-major (B), 16-bit payloads; d: 64 lanes x 16 floats.
// Lane l supplies A[l % 32][8 * (l / 32) + j] and B[8 * (l / 32) + j][l % 32] for j = 0..7 (the
// operand layout the flash kernels load K rows and Q^T columns in) and stores its 16 accumulator
// registers of D = A * B in order.
extern "C" __global__ __launch_bounds__(64) void nc_probe_mfma32x32x16(const uint16_t *a, const uint16_t *b,
                                                                        float *d, int bf16) {
    const int l = threadIdx.x;
    const int row = l % 32, k0 = 8 * (l / 32);
    u16x8 av, bv;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        av[j] = a[row * 16 + k0 + j];
        bv[j] = b[(k0 + j) * 32 + row];
    }
    floatx16 acc = {};
    if (bf16)
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, av), __builtin_bit_cast(bf16x8, bv),
                                                       acc, 0, 0, 0);
    else
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, av), __builtin_bit_cast(half8, bv), acc,
                                                      0, 0, 0);
#pragma unroll
    for (int r = 0; r < 16; ++r) d[l * 16 + r] = acc[r];
}

// LDS holds a 16 x 64 tile of 16-bit values, element (row, col) = row * 64 + col. In 16-lane group
// g = l / 16, lane m = l % 16 points at (4g + m / 4, 8g + 4 (m % 4)) — the address pattern of the
// flash kernels' V^T reads — and out[l * 4 + j] receives the j-th 16-bit value the lane gets back.
extern "C" __global__ __launch_bounds__(64) void nc_probe_ds_read_tr(uint16_t *out) {
    __shared__ __attribute__((aligned(16))) uint16_t tile[16 * 64];
    const int l = threadIdx.x;
    for (int i = l; i < 16 * 64; i += 64) tile[i] = (uint16_t)i;
    __syncthreads();
    const int g = l / 16, m = l % 16;
    const uint32_t addr = (uint32_t)(uintptr_t)tile + (uint32_t)(((4 * g + m / 4) * 64 + 8 * g + 4 * (m % 4)) * 2);
    u32x2 v;
    asm volatile("ds_read_b64_tr_b16 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=v"(v) : "v"(addr) : "memory");
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        out[l * 4 + 2 * j] = (uint16_t)(v[j] & 0xffffu);
        out[l * 4 + 2 * j + 1] = (uint16_t)(v[j] >> 16);
    }
}

// out[l * 2 + 0/1] = the two results of v_permlane32_swap(x, x) with x = 1000 + lane, in the form
// the kernels' pair_max / pair_sum consume them.
extern "C" __global__ __launch_bounds__(64) void nc_probe_permlane32(uint32_t *out) {
    const uint32_t x = 1000u + threadIdx.x;
    auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    out[threadIdx.x * 2] = r[0];
    out[threadIdx.x * 2 + 1] = r[1];
}

namespace {
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
}  // namespace

// v_mfma_scale_f32_16x16x128_f8f6f4 with A in 4 bits (e2m1) and B in 8 (e4m3), as the 4-bit cache's attention uses it.
// a: 16 rows of 64 bytes (two values a byte, the first in the low half), as_: 16 x 4 scale bytes 2^(byte - 127) of 32
// values each; b: 16 columns of 128 bytes, bs: 16 x 4. Of g = l / 16, lane l supplies values 32 g..+31 of row l % 16 of A, but
// values 16 g..+15 and 64 + 16 g..+15 of column l % 16 of B; its scales are those of values 32 g..+31 of both. It stores its 4
// accumulator registers.
extern "C" __global__ __launch_bounds__(64) void nc_probe_mfma_fp4_fp8(const uint8_t *a, const uint8_t *as_, const uint8_t *b,
                                                                        const uint8_t *bs, float *d) {
    const int l = threadIdx.x, c = l % 16, g = l / 16;
    const i32x4 x = *reinterpret_cast<const i32x4 *>(a + c * 64 + 16 * g);
    const i32x4 y0 = *reinterpret_cast<const i32x4 *>(b + c * 128 + 16 * g);
    const i32x4 y1 = *reinterpret_cast<const i32x4 *>(b + c * 128 + 64 + 16 * g);
    const i32x8 y = {y0[0], y0[1], y0[2], y0[3], y1[0], y1[1], y1[2], y1[3]};
    const i32x8 w = {x[0], x[1], x[2], x[3], 0, 0, 0, 0};
    floatx4 acc = {0.f, 0.f, 0.f, 0.f};
    acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, y, acc, 4, 0, 0, as_[c * 4 + g], 0, bs[c * 4 + g]);
#pragma unroll
    for (int r = 0; r < 4; ++r) d[l * 4 + r] = acc[r];
}

// The conversions of the 4-bit cache, a word a lane of `n`: words of 8 codes times a scale (f32, a power of two) to 8
// bf16, and of 8 f32 over the scale to a word of codes.
extern "C" __global__ __launch_bounds__(64) void nc_probe_fp4_convert(const uint32_t *codes, const float *scales, uint32_t *to_bf16,
                                                                       const float *x, uint32_t *to_codes, uint32_t n) {
    for (uint32_t i = threadIdx.x; i < n; i += 64) {
        const uint32_t w = codes[i];
        const float s = scales[i];
        to_bf16[4 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0));
        to_bf16[4 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1));
        to_bf16[4 * i + 2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2));
        to_bf16[4 * i + 3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3));
        const float *y = x + 8 * i;
        uint32_t q = 0;
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, y[0], y[1], s, 0);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, y[2], y[3], s, 1);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, y[4], y[5], s, 2);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, y[6], y[7], s, 3);
        to_codes[i] = q;
    }
}

// Pairs of f32 to e4m3 bytes and back: out[3 i] the bytes (in the low half), out[3 i + 1..2] their values.
extern "C" __global__ __launch_bounds__(64) void nc_probe_fp8_convert(const float *x, uint32_t *out, uint32_t n) {
    for (uint32_t i = threadIdx.x; i < n; i += 64) {
        const int q = __builtin_amdgcn_cvt_pk_fp8_f32(x[2 * i], x[2 * i + 1], 0, false);
        const auto y = __builtin_amdgcn_cvt_pk_f32_fp8(q, false);
        out[3 * i] = (uint32_t)q;
        out[3 * i + 1] = __builtin_bit_cast(uint32_t, (float)y[0]);
        out[3 * i + 2] = __builtin_bit_cast(uint32_t, (float)y[1]);
    }
}

// The same product with B in 6 bits (e2m3): lane l supplies values 32 g..+31 of column l % 16, 6 words of codes one after the other from the
// lowest bit up. b: 16 columns of 4 x 6 words.
extern "C" __global__ __launch_bounds__(64) void nc_probe_mfma_fp4_fp6(const uint8_t *a, const uint8_t *as_, const uint32_t *b,
                                                                        const uint8_t *bs, float *d) {
    const int l = threadIdx.x, c = l % 16, g = l / 16;
    const i32x4 x = *reinterpret_cast<const i32x4 *>(a + c * 64 + 16 * g);
    const uint32_t *y = b + (c * 4 + g) * 6;
    const i32x8 v = {(int)y[0], (int)y[1], (int)y[2], (int)y[3], (int)y[4], (int)y[5], 0, 0};
    const i32x8 w = {x[0], x[1], x[2], x[3], 0, 0, 0, 0};
    floatx4 acc = {0.f, 0.f, 0.f, 0.f};
    acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, v, acc, 4, 2, 0, as_[c * 4 + g], 0, bs[c * 4 + g]);
#pragma unroll
    for (int r = 0; r < 4; ++r) d[l * 4 + r] = acc[r];
}

// 32 f32 over a scale to 6 words of e2m3 codes, and those times the scale back: `n` such, one a thread. The first operand's 16 values are the
// even ones, the second's the odd ones.
extern "C" __global__ __launch_bounds__(64) void nc_probe_fp6_convert(const float *x, const float *scales, uint32_t *codes, float *back, uint32_t n) {
    typedef float floatx16 __attribute__((ext_vector_type(16)));
    for (uint32_t i = threadIdx.x; i < n; i += 64) {
        floatx16 even, odd;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            even[j] = x[32 * i + 2 * j];
            odd[j] = x[32 * i + 2 * j + 1];
        }
        const auto q = __builtin_amdgcn_cvt_scalef32_2xpk16_fp6_f32(even, odd, scales[i]);
        const auto y = __builtin_amdgcn_cvt_scalef32_pk32_f32_fp6(q, scales[i]);
#pragma unroll
        for (int j = 0; j < 6; ++j) codes[6 * i + j] = q[j];
#pragma unroll
        for (int j = 0; j < 32; ++j) back[32 * i + j] = y[j];
    }
}

// Four f32 over a scale to a word of e4m3 bytes, and those times the scale back.
extern "C" __global__ __launch_bounds__(64) void nc_probe_fp8_scaled(const float *x, const float *scales, uint32_t *codes, float *back, uint32_t n) {
    typedef short shortx2 __attribute__((ext_vector_type(2)));
    for (uint32_t i = threadIdx.x; i < n; i += 64) {
        const float s = scales[i];
        shortx2 q = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(shortx2{0, 0}, x[4 * i], x[4 * i + 1], s, false);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(q, x[4 * i + 2], x[4 * i + 3], s, true);
        const uint32_t w = __builtin_bit_cast(uint32_t, q);
        const auto lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, s, false), hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, s, true);
        codes[i] = w;
        back[4 * i] = lo[0];
        back[4 * i + 1] = lo[1];
        back[4 * i + 2] = hi[0];
        back[4 * i + 3] = hi[1];
    }
}
