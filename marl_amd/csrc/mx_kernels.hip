// 4-bit microscaled floating point (MXFP4): quantisation and the product of a policy layer, for gfx950.
//
//   block of 32 values x along a row:  e = max(floor(log2 max|x|) - 2, -126),  code = nearest e2m1 value of x / 2^e
//   (0, .5, 1, 1.5, 2, 3, 4, 6 and negatives; ties to the even code, above 6 to 6), scale byte e + 127;
//   a block that holds an infinity or a NaN gets scale byte 255 and reads as NaN throughout.
//   y[m][n] = sum_k x[m][k] w[n][k] + bias[n], ReLU if asked; both operands in that form, sums in float32.
//
// The scale rule is the one of the microscaling formats' specification: a block's largest value lies in [4, 8) of its
// scale, and what is above 6 becomes 6.
#include "lowbit.h"

namespace oc {

typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int MX_FP4 = 4;  // operand format code of the scaled matrix instruction: e2m1

// scale byte of a block from the bits of its largest |x|
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t top) {
    const uint32_t e = top >> 23;
    return e == 255u ? 255u : e > 3u ? e - 2u : 1u;
}

// eight codes, low nibble first; v_cvt_scalef32_pk_fp4_f32 divides by the scale, rounds to nearest even and saturates
__device__ __forceinline__ uint32_t mx_codes(const float (&v)[8], uint32_t byte) {
    const float s = bits_f(byte << 23);
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], s, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], s, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], s, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], s, 3);
    return byte == 255u ? 0u : c;
}

// ---------------------------------------------------------------------------------------------- quantise / read back

// Four lanes per block, eight values each: the block's maximum is two DPP moves away and a wave reads 2 KiB of a row in
// consecutive pieces.  Bound by memory: 131072 x 202 float32 values in 26.9 us, 4.5 TB/s (a device copy: 5.2), with 22.2 us to
// read them back, whose input is still in the last-level cache.
template <int TYPE, bool NT>
__global__ void __launch_bounds__(256)
mx_quantize_kernel(const void* __restrict__ x, int64_t rows, int cols, int64_t pitch, int blocks,
                   uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    int64_t row;
    int b, quarter;
    split_block(blockIdx.x * 256 + threadIdx.x, (uint32_t)blocks, row, b, quarter);
    if (row >= rows) return;  // whole quads leave together
    float v[8];
    load_eight<TYPE, NT>(x, row * pitch + (int64_t)b * LB_BLOCK + quarter * 8, row * pitch + cols, v);
    const uint32_t byte = mx_scale_byte(quad_max(abs_top(v)));
    reinterpret_cast<uint32_t*>(codes)[(row * blocks + b) * 4 + quarter] = mx_codes(v, byte);
    if (quarter == 0) scales[row * blocks + b] = (uint8_t)byte;
}

template <int TYPE>
__global__ void __launch_bounds__(256)
mx_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t rows, int cols,
                     int blocks, void* __restrict__ out) {
    int64_t row;
    int b, quarter;
    split_block(blockIdx.x * 256 + threadIdx.x, (uint32_t)blocks, row, b, quarter);
    if (row >= rows) return;
    const uint32_t c = reinterpret_cast<const uint32_t*>(codes)[(row * blocks + b) * 4 + quarter];
    const float s = scale_value(scales[row * blocks + b]);
    float v[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        f32x2 p;
        if (k == 0) p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 0);
        else if (k == 1) p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 1);
        else if (k == 2) p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 2);
        else p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 3);
        v[2 * k] = p.x * s;
        v[2 * k + 1] = p.y * s;
    }
    store_eight<TYPE>(out, row * cols + (int64_t)b * LB_BLOCK + quarter * 8, row * cols + cols, v);
}

// ------------------------------------------------------------------------------------------------------ the product
//
// v_mfma_scale_f32_16x16x128_f8f6f4 takes 16 rows of 128 values from each operand; lane l holds row l % 16, block l / 16
// of the four 32-value blocks, so a lane's 16 bytes of codes and its scale byte are exactly one stored block: fragments
// need no rearrangement, neither from memory nor from LDS.  The weight is the first operand, so a lane's four results
// are four output features of one row.  Rows of the weight are dealt to a wave's four tiles such that a lane has `span`
// neighbouring features, 16 bytes of float32 (4) or of a 16-bit type (8), half a block of MXFP4 (16), and the four lanes
// of a row write 64 neighbouring bytes with one store.

struct MxLinear {
    const void* x;            // float rows, or codes
    const uint8_t* x_scales;  // of codes
    int64_t rows, pitch;      // pitch in elements, float rows only
    int cols, blocks;
    const uint8_t* w;
    const uint8_t* w_scales;
    int out;                  // output features
    const float* bias;        // or NULL
    int relu;
    void* y;
    uint8_t* y_scales;        // MXFP4 output only
    float* part;              // [splits][rows][out] sums of the row's shares
    int splits;
};

// NT tiles of 16 features to a wave, 4 or 2
template <int OUT, int NT> constexpr int mx_span() {
    constexpr int most = OUT == MARL_F32 ? 4 : OUT == MARL_MXFP4 ? 16 : 8;
    return most < 4 * NT ? most : 4 * NT;
}
// first of the four neighbouring features that lane group g has from tile t
template <int OUT, int NT> __device__ __forceinline__ int mx_feature(int t, int g) {
    constexpr int SPAN = mx_span<OUT, NT>(), TILES = SPAN / 4;
    return t / TILES * (4 * SPAN) + g * SPAN + t % TILES * 4;
}

__device__ __forceinline__ f32x4 mx_mfma(u32x4 a, u32x4 b, f32x4 c, int ks, int sa, int sb) {
    const i32x8 A = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0};
    const i32x8 B = {(int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0};
    switch (ks) {  // a constant after unrolling: which byte of the scale words is used
        case 0: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, B, c, MX_FP4, MX_FP4, 0, sa, 0, sb);
        case 1: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, B, c, MX_FP4, MX_FP4, 1, sa, 1, sb);
        case 2: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, B, c, MX_FP4, MX_FP4, 2, sa, 2, sb);
        default: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, B, c, MX_FP4, MX_FP4, 3, sa, 3, sb);
    }
}

// Results of one lane: row m, v[4 t + i] is feature n0 + mx_feature(t, g) + i.  All lanes of the wave come here together
// (the MXFP4 form exchanges maxima between lanes); `live` says whether row m exists.
template <int OUT, int NT>
__device__ __forceinline__ void mx_store(const MxLinear& P, int64_t m, bool live, int n0, int g, float (&v)[4 * NT]) {
    constexpr int SPAN = mx_span<OUT, NT>();
    if (P.relu) {
#pragma unroll
        for (int k = 0; k < 4 * NT; ++k) v[k] = v[k] < 0.0f ? 0.0f : v[k];  // a NaN stays
    }
    if constexpr (OUT == MARL_MXFP4) {
        const int n = n0 + SPAN * g;
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < SPAN; ++k) {
            if (n + k >= P.out) v[k] = 0.0f;
            top = max(top, f_bits(v[k]) & 0x7FFFFFFFu);
        }
        top = max(top, (uint32_t)__shfl_xor((int)top, 16, 64));  // the lanes with the rest of the block
        if constexpr (NT == 2) top = max(top, (uint32_t)__shfl_xor((int)top, 32, 64));
        const int yb = (P.out + LB_BLOCK - 1) / LB_BLOCK, b = n / LB_BLOCK;
        if (!live || b >= yb) return;
        const uint32_t byte = mx_scale_byte(top);
        uint32_t* to = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(P.y) + (m * yb + b) * 16 + (n & (LB_BLOCK - 1)) / 2);
        float part[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) part[k] = v[k];
        if constexpr (SPAN == 16) {
            float rest[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) rest[k] = v[8 + k];
            *reinterpret_cast<u32x2*>(to) = u32x2{mx_codes(part, byte), mx_codes(rest, byte)};
        } else {
            *to = mx_codes(part, byte);
        }
        if ((n & (LB_BLOCK - 1)) == 0) P.y_scales[m * yb + b] = (uint8_t)byte;
    } else {
        if (!live) return;
        const int64_t row = m * P.out;
#pragma unroll
        for (int s = 0; s < 4 * NT / SPAN; ++s) {
            const int n = n0 + mx_feature<OUT, NT>(s * SPAN / 4, g);
            if (n + SPAN <= P.out) {
                if constexpr (OUT == MARL_F32) {
                    *reinterpret_cast<f32x4_a4*>(static_cast<float*>(P.y) + row + n) = f32x4{v[4 * s], v[4 * s + 1], v[4 * s + 2], v[4 * s + 3]};
                } else {
                    u32x4 u;
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        u[k] = (uint32_t)to_half_type<OUT>(v[8 * s + 2 * k]) | (uint32_t)to_half_type<OUT>(v[8 * s + 2 * k + 1]) << 16;
                    *reinterpret_cast<u32x4_a2*>(static_cast<uint16_t*>(P.y) + row + n) = u;
                }
            } else {
#pragma unroll
                for (int k = 0; k < SPAN; ++k) {
                    if (n + k >= P.out) continue;
                    if constexpr (OUT == MARL_F32) static_cast<float*>(P.y)[row + n + k] = v[SPAN * s + k];
                    else static_cast<uint16_t*>(P.y)[row + n + k] = to_half_type<OUT>(v[SPAN * s + k]);
                }
            }
        }
    }
}

// Rows of 8 to 512 values.  A workgroup has eight waves, WN of them side by side (16 NT = 64 features each) and 8 / WN below one
// another, and walks row tiles; a wave keeps its features' whole weight in registers (at most 64 of them).  The threads
// quantise a tile's rows into LDS (four lanes per block, as above); the next tile's values are on their way from memory
// meanwhile.  Bound by memory: rows in, results out, the weight once per workgroup.  float32 rows and results: 131072 x 202 ->
// 512 in 79 us (4.7 TB/s), 131072 x 512 -> 256 in 75 us (5.4 TB/s; with MXFP4 rows 33 us).  Few rows, with 32 features to a wave and one
// tile to a workgroup, take 3 to 5 us, of which a launch is 2.
template <int WN, int NT>
struct MxTile {
    static constexpr int WM = 8 / WN, GROUPS = WN == 8 && NT == 4 ? 2 : 1;  // waves along the rows; groups of 16 rows each of them has
    static constexpr int ROWS = 16 * WM * GROUPS;
};

// eight values of a row as they come from memory; `n` of them exist
template <int TYPE> struct MxRaw { u32x4 u[TYPE == MARL_F32 ? 2 : 1]; };
template <int TYPE>
__device__ __forceinline__ void raw_load(MxRaw<TYPE>& raw, const void* x, int64_t at) {
    if constexpr (TYPE == MARL_F32) {
        typedef u32x4 u32x4_a4 __attribute__((aligned(4)));
        const u32x4_a4* p = reinterpret_cast<const u32x4_a4*>(static_cast<const uint32_t*>(x) + at);
        raw.u[0] = p[0];
        raw.u[1] = p[1];
    } else {
        raw.u[0] = *reinterpret_cast<const u32x4_a2*>(static_cast<const uint16_t*>(x) + at);
    }
}
template <int TYPE>
__device__ __forceinline__ void raw_use(const MxRaw<TYPE>& raw, float (&v)[8]) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        if constexpr (TYPE == MARL_F32) v[k] = bits_f(raw.u[k >> 2][k & 3]);
        else if constexpr (TYPE == MARL_BF16) v[k] = bits_f(k & 1 ? raw.u[0][k >> 1] & 0xFFFF0000u : raw.u[0][k >> 1] << 16);
        else v[k] = k & 1 ? half_hi(raw.u[0][k >> 1]) : half_lo(raw.u[0][k >> 1]);
    }
}

// Workgroups on a compute unit.  Two where a wave has two tiles of features, and for MXFP4 results of float rows, which are small and
// leave the quantising, if the registers suffice (131072 x 202 -> 512 in float32: 48 against 42 us; not with 16 blocks a row, 59
// and 65 us, nor with the 64 rows that two waves side by side have, 24 and 28).  Elsewhere two read the weight twice and are slower
// (131072 x 512 -> 256 from MXFP4 to MXFP4 27 and 35 us).
constexpr int mx_workgroups(int ks, int in, int out, int wn, int nt) {
    return nt == 2 || (out == MARL_MXFP4 && in != MARL_MXFP4 && ks == 2 && wn > 2) ? 2 : 1;
}

// ONE: a workgroup has one tile
template <int KS, int IN, int OUT, int WN, int NT, bool ONE>
__global__ void __launch_bounds__(512, 2 * mx_workgroups(KS, IN, OUT, WN, NT))
mx_rows_kernel(MxLinear P) {
    typedef MxTile<WN, NT> T;
    constexpr int NB = KS * 4;             // blocks of a row, padded to whole matrix instructions
    constexpr int PITCH = NB * 16 + 16;    // LDS bytes per row of codes; the 16 keep a wave's rows apart in the banks
    constexpr int ITEMS = T::ROWS * NB * (IN == MARL_MXFP4 ? 1 : 4) / 512 > 0 ? T::ROWS * NB * (IN == MARL_MXFP4 ? 1 : 4) / 512 : 1;
    static_assert(ITEMS <= 4, "the next tile's values are in registers meanwhile");
    // Whether the next tile is filled in before this one is multiplied, and loads go out two tiles earlier: a store does not
    // hold up the loads behind it then.  131072 rows: MXFP4 512 -> 256 in 32.5 us, otherwise 37; float32 202 -> 512 80 and 82.
    // It takes registers: MXFP4 results of float rows, which live on two workgroups a compute unit, 45 and 42.
    constexpr bool PIPED = NT == 4 && (IN == MARL_MXFP4 || (IN == MARL_F32 && OUT != MARL_MXFP4 && WN > 2));
    __shared__ __align__(16) uint8_t codes[2][T::ROWS][PITCH];
    __shared__ __align__(16) uint8_t scales[2][T::ROWS][16];  // [block % 4][block / 4]: a lane's scales are one word
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 15, g = lane >> 4;
    const int n0 = (blockIdx.y * WN + wave % WN) * (16 * NT), wm = wave / WN * 16 * T::GROUPS;
    // Features behind the last are the last again (their results are not stored), blocks behind a row's end its last one again
    // (x is zero there): no load hangs on a condition, so that all of them are under way together.
    u32x4 w[NT][KS];
    uint32_t wsb[NT][KS];
    float bias[4 * NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int64_t row = (int64_t)min(n0 + mx_feature<OUT, NT>(t, r >> 2) + (r & 3), P.out - 1) * P.blocks;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const int64_t at = row + min(ks * 4 + g, P.blocks - 1);
            w[t][ks] = *reinterpret_cast<const u32x4*>(P.w + at * 16);
            wsb[t][ks] = P.w_scales[at];
        }
    }
    if (P.bias) {
#pragma unroll
        for (int k = 0; k < 4 * NT; ++k) bias[k] = P.bias[min(n0 + mx_feature<OUT, NT>(k >> 2, g) + (k & 3), P.out - 1)];
    } else {
#pragma unroll
        for (int k = 0; k < 4 * NT; ++k) bias[k] = 0.0f;
    }

    // An item: 8 values of a block (float rows) or a whole block (codes).  Rows behind the last are the last again, their
    // results are not stored; every path makes the same loads.
    const int64_t all = (P.rows - 1) * P.pitch + P.cols;  // elements from the first row's start to the last one's end
    MxRaw<IN == MARL_MXFP4 ? MARL_BF16 : IN> raw[PIPED ? 2 : 1][ITEMS];
    uint32_t raw_s[PIPED ? 2 : 1][ITEMS];
    const auto load = [&](int64_t tile, int q, int set, int slot) {
        const int it = tid + q * 512;
        if constexpr (IN == MARL_MXFP4) {
            const int64_t m = min(tile * T::ROWS + it / NB, P.rows - 1) * P.blocks + min(it % NB, P.blocks - 1);
            raw[set][slot].u[0] = reinterpret_cast<const u32x4*>(P.x)[m];
            raw_s[set][slot] = P.x_scales[m];
        } else {
            const int64_t m = min(tile * T::ROWS + (it >> 2) / NB, P.rows - 1);
            raw_load<IN>(raw[set][slot], P.x, min(m * P.pitch + (it >> 2) % NB * LB_BLOCK + (it & 3) * 8, all - 8));
        }
    };
    const auto quantise = [&](int64_t tile, int q, int set, int slot, int buf) {
        const int it = tid + q * 512;
        if (T::ROWS * NB * (IN == MARL_MXFP4 ? 1 : 4) < 512 && it >= T::ROWS * NB * (IN == MARL_MXFP4 ? 1 : 4)) return;
        if constexpr (IN == MARL_MXFP4) {
            const int row = it / NB, b = it % NB;
            const bool there = b < P.blocks;
            *reinterpret_cast<u32x4*>(&codes[buf][row][b * 16]) = there ? raw[set][slot].u[0] : u32x4{0, 0, 0, 0};
            scales[buf][row][(b & 3) * 4 + (b >> 2)] = (uint8_t)(there ? raw_s[set][slot] : 127u);
        } else {
            const int quarter = it & 3, b = (it >> 2) % NB, row = (it >> 2) / NB;
            float v[8];
            raw_use<IN>(raw[set][slot], v);
            // What lies behind a row's end is the next row, and counts as 0; only behind the last row there is nothing, and
            // its last values were read as the tensor's last eight: move them down.
            const int64_t back = min(tile * T::ROWS + row, P.rows - 1) * P.pitch + b * LB_BLOCK + quarter * 8 - (all - 8);
            if (back > 0) {
#pragma unroll
                for (int step = 4; step >= 1; step >>= 1)
#pragma unroll
                    for (int k = 0; k < 8; ++k) v[k] = back & step ? (k + step < 8 ? v[k + step] : 0.0f) : v[k];
            }
            const int n = P.cols - b * LB_BLOCK - quarter * 8;  // how many of the eight exist
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = k < n ? v[k] : 0.0f;
            const uint32_t byte = mx_scale_byte(quad_max(abs_top(v)));
            *reinterpret_cast<uint32_t*>(&codes[buf][row][b * 16 + quarter * 4]) = mx_codes(v, byte);
            if (quarter == 0) scales[buf][row][(b & 3) * 4 + (b >> 2)] = (uint8_t)byte;
        }
    };

    const int64_t tiles = (P.rows + T::ROWS - 1) / T::ROWS, step = gridDim.x;
#pragma unroll
    for (int set = 0; set < (PIPED ? 2 : 1); ++set)
#pragma unroll
        for (int q = 0; q < ITEMS; ++q) load(blockIdx.x + set * step, q, set, q);
    int ws[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        uint32_t word = 0;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) word |= wsb[t][ks] << (8 * ks);
        ws[t] = (int)word;
    }
    const auto multiply = [&](int64_t tile, int buf) {
#pragma unroll
        for (int rt = 0; rt < T::GROUPS; ++rt) {
            f32x4 acc[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) acc[t] = f32x4{0, 0, 0, 0};
            const int row = wm + rt * 16 + r;
            const int xs = *reinterpret_cast<const int*>(&scales[buf][row][g * 4]);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const u32x4 x = *reinterpret_cast<const u32x4*>(&codes[buf][row][(ks * 4 + g) * 16]);
#pragma unroll
                for (int t = 0; t < NT; ++t) acc[t] = mx_mfma(w[t][ks], x, acc[t], ks, ws[t], xs);
            }
            float v[4 * NT];
#pragma unroll
            for (int k = 0; k < 4 * NT; ++k) v[k] = acc[k >> 2][k & 3] + bias[k];
            const int64_t m = tile * T::ROWS + row;
            mx_store<OUT, NT>(P, m, m < P.rows, n0, g, v);
        }
    };
    // One barrier a tile: the other buffer is free once every wave has come there.
    if constexpr (PIPED) {
        // a tile's values, loaded into raw[set], into LDS buffer `buf`, and the loads of the next tile for that set
        const auto fill = [&](int64_t tile, int buf, int set) {
#pragma unroll
            for (int q = 0; q < ITEMS; ++q) quantise(tile, q, set, q, buf);
#pragma unroll
            for (int q = 0; q < ITEMS; ++q) load(tile + 2 * step, q, set, q);
        };
        fill(blockIdx.x, 0, 0);
        __syncthreads();
        for (int64_t tile = blockIdx.x; tile < tiles; tile += 2 * step) {
            if (tile + step < tiles) fill(tile + step, 1, 1);
            multiply(tile, 0);
            __syncthreads();
            if (tile + step >= tiles) break;
            if (tile + 2 * step < tiles) fill(tile + 2 * step, 0, 0);
            multiply(tile + step, 1);
            __syncthreads();
        }
    } else if constexpr (ONE) {
#pragma unroll
        for (int q = 0; q < ITEMS; ++q) quantise(blockIdx.x, q, 0, q, 0);
        __syncthreads();
        multiply(blockIdx.x, 0);
    } else {
        int buf = 0;
        for (int64_t tile = blockIdx.x; tile < tiles; tile += step, buf ^= 1) {
#pragma unroll
            for (int q = 0; q < ITEMS; ++q) {
                quantise(tile, q, 0, q, buf);
                load(tile + step, q, 0, q);
            }
            __syncthreads();
            multiply(tile, buf);
        }
    }
}

// Up to 16 rows of any length (a joint observation): the weight, read once, is what such a call costs.  A workgroup has 16
// features and a share of the row (grid y), its four waves every fourth chunk of 2048 values each, whose 64 loads of 1 KiB
// are under way together; the sums of the shares are joined by mx_join_kernel.
// Which block goes to which matrix instruction is free as long as both operands agree: of a stretch of 512 values lane group
// g has blocks 4 g .. 4 g + 3, so that a lane reads 64 neighbouring bytes of codes and its four scales as one word, and the
// four lanes of a row 256 bytes, a wave 1 KiB of each of its 16 rows.  (With 64 features to a wave and 256 bytes of each row
// at a time, 1 x 827392 -> 512 took 57 us.)  Bound by memory: that product in 48 us, 4.7 TB/s, behind 5 us for quantising x
// and before 5 us for the sums.  The non-temporal hint costs it half as much again: the four lanes of a row share lines.
struct MxStretch { u32x4 c[4]; uint32_t s; };
__device__ __forceinline__ void load_stretch(MxStretch& v, const uint8_t* codes, const uint8_t* scales, int64_t at) {
    v.s = *reinterpret_cast<const u32_a1*>(scales + at);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) v.c[ks] = *reinterpret_cast<const u32x4*>(codes + (at + ks) * 16);
}
// a row's last stretch: block b + ks of `blocks`, those behind the end are the last one again, and zeros if `zero`
__device__ __forceinline__ void load_last_stretch(MxStretch& v, const uint8_t* codes, const uint8_t* scales, int64_t row, int b, int blocks, bool zero) {
    v.s = 0;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
        const bool there = b + ks < blocks || !zero;
        const int64_t at = row + min(b + ks, blocks - 1);
        const u32x4 c = *reinterpret_cast<const u32x4*>(codes + at * 16);
        v.c[ks] = there ? c : u32x4{0, 0, 0, 0};
        v.s |= (there ? (uint32_t)scales[at] : 127u) << (8 * ks);
    }
}

__global__ void __launch_bounds__(256, 2)
mx_few_rows_kernel(MxLinear P) {
    __shared__ f32x4 sums[3][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * 16;
    const int chunks = (P.blocks + 63) / 64, per = (chunks + P.splits - 1) / P.splits;
    const int first = blockIdx.y * per, last = min(chunks, first + per);
    const int64_t wrow = (int64_t)min(n0 + r, P.out - 1) * P.blocks, xrow = min((int64_t)r, P.rows - 1) * P.blocks;
    const uint8_t* xc = static_cast<const uint8_t*>(P.x);
    f32x4 acc[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) acc[u] = f32x4{0, 0, 0, 0};
    for (int c = first + wave; c < last; c += 4) {
        MxStretch w[4], x[4];
        const int b = c * 64 + 4 * g;
        if (c * 64 + 64 <= P.blocks) {
#pragma unroll
            for (int u = 0; u < 4; ++u) load_stretch(w[u], P.w, P.w_scales, wrow + b + 16 * u);
#pragma unroll
            for (int u = 0; u < 4; ++u) load_stretch(x[u], xc, P.x_scales, xrow + b + 16 * u);
        } else {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                load_last_stretch(w[u], P.w, P.w_scales, wrow, b + 16 * u, P.blocks, false);
                load_last_stretch(x[u], xc, P.x_scales, xrow, b + 16 * u, P.blocks, true);
            }
        }
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
#pragma unroll
            for (int u = 0; u < 4; ++u) acc[u] = mx_mfma(w[u].c[ks], x[u].c[ks], acc[u], ks, (int)w[u].s, (int)x[u].s);
    }
    f32x4 v = (acc[0] + acc[1]) + (acc[2] + acc[3]);
    if (wave) sums[wave - 1][lane] = v;
    __syncthreads();
    if (wave || r >= P.rows) return;
    v = (v + sums[0][lane]) + (sums[1][lane] + sums[2][lane]);
    float* part = P.part + ((int64_t)blockIdx.y * P.rows + r) * P.out + n0 + 4 * g;
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (n0 + 4 * g + k < P.out) part[k] = v[k];
}

// More rows of any length: 64 features and 64 rows to a workgroup, whose four waves take every fourth stretch of 512 values
// each and add their sums through LDS; with few workgroups the row is split over them too (grid z).  Fragments come straight
// from the caches, four waves reading the same lines: 4096 x 4096 -> 4096 in 165 us, 0.83 PFLOP/s.
constexpr int MX_RM = 4;  // groups of 16 rows
template <int OUT>
__global__ void __launch_bounds__(256, 2)
mx_stream_kernel(MxLinear P) {
    constexpr int RM = MX_RM;
    __shared__ float sums[3][RM][64][17];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * 64;
    const int64_t m0 = (int64_t)blockIdx.y * (16 * RM);
    const int stretches = (P.blocks + 15) / 16, per = (stretches + P.splits - 1) / P.splits;
    const int first = blockIdx.z * per, last = min(stretches, first + per);
    f32x4 acc[RM][4];
#pragma unroll
    for (int q = 0; q < RM; ++q)
#pragma unroll
        for (int t = 0; t < 4; ++t) acc[q][t] = f32x4{0, 0, 0, 0};
    // rows and features behind the last are the last again, their results are not stored
    int64_t wrow[4], xrow[RM];
#pragma unroll
    for (int t = 0; t < 4; ++t) wrow[t] = (int64_t)min(n0 + mx_feature<OUT, 4>(t, r >> 2) + (r & 3), P.out - 1) * P.blocks;
#pragma unroll
    for (int q = 0; q < RM; ++q) xrow[q] = min(m0 + q * 16 + r, P.rows - 1) * P.blocks;
    const uint8_t* xc = static_cast<const uint8_t*>(P.x);
    for (int s = first + wave; s < last; s += 4) {
        MxStretch w[4], x[RM];
        const int b = s * 16 + 4 * g;
        if (s * 16 + 16 <= P.blocks) {
#pragma unroll
            for (int q = 0; q < RM; ++q) load_stretch(x[q], xc, P.x_scales, xrow[q] + b);
#pragma unroll
            for (int t = 0; t < 4; ++t) load_stretch(w[t], P.w, P.w_scales, wrow[t] + b);
        } else {
#pragma unroll
            for (int q = 0; q < RM; ++q) load_last_stretch(x[q], xc, P.x_scales, xrow[q], b, P.blocks, true);
#pragma unroll
            for (int t = 0; t < 4; ++t) load_last_stretch(w[t], P.w, P.w_scales, wrow[t], b, P.blocks, false);
        }
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
#pragma unroll
            for (int q = 0; q < RM; ++q)
#pragma unroll
                for (int t = 0; t < 4; ++t) acc[q][t] = mx_mfma(w[t].c[ks], x[q].c[ks], acc[q][t], ks, (int)w[t].s, (int)x[q].s);
    }
    if (wave) {
#pragma unroll
        for (int q = 0; q < RM; ++q)
#pragma unroll
            for (int k = 0; k < 16; ++k) sums[wave - 1][q][lane][k] = acc[q][k >> 2][k & 3];
    }
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int q = 0; q < RM; ++q) {
        float v[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) v[k] = ((acc[q][k >> 2][k & 3] + sums[0][q][lane][k]) + sums[1][q][lane][k]) + sums[2][q][lane][k];
        const int64_t m = m0 + q * 16 + r;
        if (P.splits > 1) {
            if (m >= P.rows) continue;
            float* part = P.part + ((int64_t)blockIdx.z * P.rows + m) * P.out;
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                const int n = n0 + mx_feature<OUT, 4>(k >> 2, g) + (k & 3);
                if (n < P.out) part[n] = v[k];
            }
        } else {
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                const int n = n0 + mx_feature<OUT, 4>(k >> 2, g) + (k & 3);
                v[k] += P.bias && n < P.out ? P.bias[n] : 0.0f;
            }
            mx_store<OUT, 4>(P, m, m < P.rows, n0, g, v);
        }
    }
}

// Sums of the splits, then bias, ReLU and the output's type.  Four lanes per 32 features, as in quantising; a workgroup's
// four waves have every fourth split each, and their four sums are added in order.
template <int OUT>
__global__ void __launch_bounds__(256)
mx_join_kernel(MxLinear P) {
    __shared__ float sums[3][8][64];
    const int yb = (P.out + LB_BLOCK - 1) / LB_BLOCK, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int64_t m;
    int b, quarter;
    split_block(blockIdx.x * 64 + lane, (uint32_t)yb, m, b, quarter);
    const int n = b * LB_BLOCK + quarter * 8;
    const bool live = m < P.rows && n < P.out;
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = 0.0f;
    if (live) {
        const int64_t step = P.rows * P.out;
#pragma unroll 4
        for (int s = wave; s < P.splits; s += 4) {
            float p[8];
            load_eight<MARL_F32>(P.part, s * step + m * P.out + n, s * step + m * P.out + P.out, p);
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] += p[k];
        }
    }
    if (wave) {
#pragma unroll
        for (int k = 0; k < 8; ++k) sums[wave - 1][k][lane] = v[k];
    }
    __syncthreads();
    if (wave || m >= P.rows) return;  // whole quads leave together
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        v[k] = (v[k] + sums[0][k][lane]) + (sums[1][k][lane] + sums[2][k][lane]);
        if (n + k >= P.out) { v[k] = 0.0f; continue; }
        if (P.bias) v[k] += P.bias[n + k];
        if (P.relu) v[k] = v[k] < 0.0f ? 0.0f : v[k];
    }
    if constexpr (OUT == MARL_MXFP4) {
        const uint32_t byte = mx_scale_byte(quad_max(abs_top(v)));
        reinterpret_cast<uint32_t*>(P.y)[(m * yb + b) * 4 + quarter] = mx_codes(v, byte);
        if (quarter == 0) P.y_scales[m * yb + b] = (uint8_t)byte;
    } else if (n < P.out) {
        store_eight<OUT>(P.y, m * P.out + n, m * P.out + P.out, v);
    }
}

// ------------------------------------------------------------------------------------------------------------ host

// rows that mx_rows_kernel takes: its loads are eight values wide, its weight registers hold four matrix instructions
static bool mx_short_rows(int64_t cols) { return cols >= 8 && cols <= 512; }

static hipError_t launch_quantize(const void* x, int type, int64_t rows, int cols, int64_t pitch, uint8_t* codes,
                                  uint8_t* scales, hipStream_t stream) {
    const int blocks = (int)lb_blocks(cols);
    const bool nt = (uint64_t)rows * cols * lb_type_bytes(type) > LB_NT_BYTES;
    auto kernel = type == MARL_F32 ? (nt ? mx_quantize_kernel<MARL_F32, true> : mx_quantize_kernel<MARL_F32, false>)
                : type == MARL_BF16 ? (nt ? mx_quantize_kernel<MARL_BF16, true> : mx_quantize_kernel<MARL_BF16, false>)
                                    : (nt ? mx_quantize_kernel<MARL_F16, true> : mx_quantize_kernel<MARL_F16, false>);
    hipLaunchKernelGGL(kernel, dim3(block_grid(rows, cols)), dim3(256), 0, stream, x, rows, cols, pitch, blocks, codes, scales);
    return hipGetLastError();
}

template <int KS, int IN, int WN, int NT, bool ONE>
static void (*rows_kernel_out(int out))(MxLinear) {
    switch (out) {
        case MARL_F32: return mx_rows_kernel<KS, IN, MARL_F32, WN, NT, ONE>;
        case MARL_BF16: return mx_rows_kernel<KS, IN, MARL_BF16, WN, NT, ONE>;
        case MARL_F16: return mx_rows_kernel<KS, IN, MARL_F16, WN, NT, ONE>;
        default: return mx_rows_kernel<KS, IN, MARL_MXFP4, WN, NT, ONE>;
    }
}
// FLOATS, CODES: which rows come here
template <int KS, int WN, int NT, bool ONE, bool FLOATS, bool CODES>
static void launch_rows(const MxLinear& P, int in, int out, hipStream_t stream) {
    void (*kernel)(MxLinear) = nullptr;
    if constexpr (FLOATS)
        kernel = in == MARL_F32 ? rows_kernel_out<KS, MARL_F32, WN, NT, ONE>(out) : in == MARL_BF16 ? rows_kernel_out<KS, MARL_BF16, WN, NT, ONE>(out)
                                                                                                    : rows_kernel_out<KS, MARL_F16, WN, NT, ONE>(out);
    if constexpr (CODES)
        if (in == MARL_MXFP4) kernel = rows_kernel_out<KS, MARL_MXFP4, WN, NT, ONE>(out);
    const int64_t tiles = (P.rows + MxTile<WN, NT>::ROWS - 1) / MxTile<WN, NT>::ROWS;
    const int64_t resident = ONE ? tiles : 256 * mx_workgroups(KS, in, out, WN, NT);
    hipLaunchKernelGGL(kernel, dim3((uint32_t)(tiles < resident ? tiles : resident), (P.out + 16 * NT * WN - 1) / (16 * NT * WN)), dim3(512), 0, stream, P);
}
template <int KS>
static void launch_rows_wide(const MxLinear& P, int in, int out, hipStream_t stream) {
    // Where tiles of 16 rows and 256 features are at most two to a compute unit, those: a wave has half the weight to fetch before it can
    // multiply, and that is what few rows take.  In us, with them and without: 202 -> 512 in float32 32 rows 3.2 and 5.8, 2048 rows
    // 3.9 and 6.5, 4096 (512 tiles) 5.8 and 7.1, 8192 9.0 and 7.9; 512 -> 256 from MXFP4 32 rows 4.5 and 8.4, 4096 5.3 and 9.1.
    const int64_t small = (P.rows + 15) / 16 * ((P.out + 255) / 256);
    if (small <= 512) return launch_rows<KS, 8, 2, true, true, true>(P, in, out, stream);
    // The same tiles, walked by two workgroups a compute unit, for long float rows whose features they cover: 131072 x 512 -> 256 in
    // float32 75 us, with four tiles of features to a wave 81; 21847 x 420 -> 250 in bfloat16 11.7 and 13.0; 131072 x 400 -> 100 48
    // and 65.  Not for short rows (131072 x 202 -> 256 45 and 45, to MXFP4 32 and 25) nor for codes (512 -> 256 37 and 33).
    if constexpr (KS == 4)
        if (in != MARL_MXFP4 && P.out <= 256) return launch_rows<KS, 8, 2, false, true, false>(P, in, out, stream);
    // Otherwise side by side as many waves as there are features for, so that a row is quantised once.
    if (P.out <= 128) launch_rows<KS, 2, 4, false, KS == 2, true>(P, in, out, stream);
    else if (P.out <= 256) launch_rows<KS, 4, 4, false, KS == 2, true>(P, in, out, stream);
    else launch_rows<KS, 8, 4, false, true, true>(P, in, out, stream);
}
static void (*stream_kernel(int out))(MxLinear) {
    switch (out) {
        case MARL_F32: return mx_stream_kernel<MARL_F32>;
        case MARL_BF16: return mx_stream_kernel<MARL_BF16>;
        case MARL_F16: return mx_stream_kernel<MARL_F16>;
        default: return mx_stream_kernel<MARL_MXFP4>;
    }
}

// How a call over other rows is cut: whether mx_few_rows_kernel takes it, and into how many shares of the row.
struct MxCut { bool few; int splits; };
constexpr int64_t MX_GROUPS = 512;  // two workgroups a compute unit
static MxCut mx_cut(int64_t rows, int64_t cols, int out) {
    MxCut c;
    c.few = rows <= 16;
    const int64_t unit = c.few ? 64 : 16, units = ((int64_t)lb_blocks(cols) + unit - 1) / unit;  // chunks, stretches
    const int64_t groups = c.few ? (out + 15) / 16 : ((out + 63) / 64) * ((rows + 16 * MX_RM - 1) / (16 * MX_RM));
    const int64_t most = units / 8 < 1 ? 1 : units / 8;  // at least two for each of a workgroup's four waves
    int64_t s = MX_GROUPS / groups;
    s = s < 1 ? 1 : s > most ? most : s;
    const int64_t per = (units + s - 1) / s;
    c.splits = (int)((units + per - 1) / per);
    return c;
}
static size_t up16(size_t n) { return (n + 15) & ~(size_t)15; }

static hipError_t launch_linear(const MxLinear& P0, int x_type, int out_type, uint8_t* ws, hipStream_t stream) {
    MxLinear P = P0;
    if (mx_short_rows(P.cols)) {
        if (P.blocks <= 8) launch_rows_wide<2>(P, x_type, out_type, stream);
        else launch_rows_wide<4>(P, x_type, out_type, stream);
        return hipGetLastError();
    }
    const MxCut c = mx_cut(P.rows, P.cols, P.out);
    if (x_type != MARL_MXFP4) {
        uint8_t* codes = ws;
        ws += up16((size_t)P.rows * P.blocks * 16);
        uint8_t* scales = ws;
        ws += up16((size_t)P.rows * P.blocks);
        hipError_t e = launch_quantize(P.x, x_type, P.rows, P.cols, P.pitch, codes, scales, stream);
        if (e != hipSuccess) return e;
        P.x = codes;
        P.x_scales = scales;
    }
    P.splits = c.splits;
    P.part = reinterpret_cast<float*>(ws);
    if (c.few)
        hipLaunchKernelGGL(mx_few_rows_kernel, dim3((P.out + 15) / 16, c.splits), dim3(256), 0, stream, P);
    else
        hipLaunchKernelGGL(stream_kernel(out_type), dim3((P.out + 63) / 64, (uint32_t)((P.rows + 16 * MX_RM - 1) / (16 * MX_RM)), c.splits),
                           dim3(256), 0, stream, P);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || (!c.few && c.splits == 1)) return e;
    auto join = out_type == MARL_F32 ? mx_join_kernel<MARL_F32> : out_type == MARL_BF16 ? mx_join_kernel<MARL_BF16>
              : out_type == MARL_F16 ? mx_join_kernel<MARL_F16> : mx_join_kernel<MARL_MXFP4>;
    hipLaunchKernelGGL(join, dim3((uint32_t)((P.rows * lb_blocks(P.out) * 4 + 63) / 64)), dim3(256), 0, stream, P);
    return hipGetLastError();
}

static int hip_result(hipError_t e, const char* what) {
    if (e == hipSuccess) return MARL_OK;
    return set_error(MARL_ERR_HIP, std::string(what) + ": " + hipGetErrorString(e));
}

}  // namespace oc

using namespace oc;

extern "C" int marl_mx_quantize(const void* d_x, int x_type, int64_t num_rows, int num_cols, int64_t row_stride,
                                uint8_t* d_codes, uint8_t* d_scales, void* stream) {
    if (num_rows < 0 || num_cols <= 0) return set_error(MARL_ERR_INVALID, "num_rows must not be negative and num_cols must be positive");
    if (x_type != MARL_F32 && x_type != MARL_BF16 && x_type != MARL_F16)
        return set_error(MARL_ERR_INVALID, "x_type must be MARL_F32, MARL_BF16 or MARL_F16");
    if (num_rows == 0) return MARL_OK;
    if (!d_x || !d_codes || !d_scales) return set_error(MARL_ERR_INVALID, "NULL argument to marl_mx_quantize");
    if (row_stride == 0) row_stride = num_cols;
    if (row_stride < num_cols) return set_error(MARL_ERR_INVALID, "row_stride is smaller than num_cols");
    if (((uintptr_t)d_x & (lb_type_bytes(x_type) - 1)) != 0 || ((uintptr_t)d_codes & 15u) != 0)
        return set_error(MARL_ERR_INVALID, "d_x must be aligned to its elements, d_codes to 16 bytes");
    if (too_many_blocks(num_rows, num_cols)) return set_error(MARL_ERR_INVALID, "more than 2^30 - 64 blocks of 32 values in one call");
    return hip_result(launch_quantize(d_x, x_type, num_rows, num_cols, row_stride, d_codes, d_scales, reinterpret_cast<hipStream_t>(stream)),
                      "MXFP4 quantisation launch");
}

extern "C" int marl_mx_dequantize(const uint8_t* d_codes, const uint8_t* d_scales, int64_t num_rows, int num_cols, int out_type,
                                  void* d_out, void* stream) {
    if (num_rows < 0 || num_cols <= 0) return set_error(MARL_ERR_INVALID, "num_rows must not be negative and num_cols must be positive");
    if (out_type != MARL_F32 && out_type != MARL_BF16 && out_type != MARL_F16)
        return set_error(MARL_ERR_INVALID, "out_type must be MARL_F32, MARL_BF16 or MARL_F16");
    if (num_rows == 0) return MARL_OK;
    if (!d_codes || !d_scales || !d_out) return set_error(MARL_ERR_INVALID, "NULL argument to marl_mx_dequantize");
    if (((uintptr_t)d_codes & 15u) != 0 || ((uintptr_t)d_out & (lb_type_bytes(out_type) - 1)) != 0)
        return set_error(MARL_ERR_INVALID, "d_codes must be 16-byte aligned, d_out aligned to its elements");
    if (too_many_blocks(num_rows, num_cols)) return set_error(MARL_ERR_INVALID, "more than 2^30 - 64 blocks of 32 values in one call");
    const int blocks = (int)lb_blocks(num_cols);
    auto kernel = out_type == MARL_F32 ? mx_dequantize_kernel<MARL_F32> : out_type == MARL_BF16 ? mx_dequantize_kernel<MARL_BF16> : mx_dequantize_kernel<MARL_F16>;
    hipLaunchKernelGGL(kernel, dim3(block_grid(num_rows, num_cols)), dim3(256), 0, reinterpret_cast<hipStream_t>(stream), d_codes, d_scales, num_rows, num_cols, blocks, d_out);
    return hip_result(hipGetLastError(), "MXFP4 read-back launch");
}

extern "C" size_t marl_mx_linear_workspace_bytes(int x_type, int64_t num_rows, int num_cols, int num_out) {
    if (num_rows <= 0 || num_cols <= 0 || mx_short_rows(num_cols) || num_out <= 0) return 0;
    const MxCut c = mx_cut(num_rows, num_cols, num_out);
    size_t n = 0;
    if (x_type != MARL_MXFP4) n += up16((size_t)num_rows * lb_blocks(num_cols) * 16) + up16((size_t)num_rows * lb_blocks(num_cols));
    if (c.few || c.splits > 1) n += (size_t)c.splits * num_rows * num_out * sizeof(float);
    return n;
}

extern "C" int marl_mx_linear(const void* d_x, const uint8_t* d_x_scales, int x_type, int64_t num_rows, int num_cols, int64_t row_stride,
                              const uint8_t* d_w_codes, const uint8_t* d_w_scales, int num_out, const float* d_bias, int relu,
                              void* d_y, uint8_t* d_y_scales, int y_type, void* d_workspace, void* stream) {
    if (num_rows < 0 || num_cols <= 0 || num_out <= 0)
        return set_error(MARL_ERR_INVALID, "num_rows must not be negative, num_cols and num_out must be positive");
    if (x_type < MARL_F32 || x_type > MARL_MXFP4 || y_type < MARL_F32 || y_type > MARL_MXFP4)
        return set_error(MARL_ERR_INVALID, "x_type and y_type must be MARL_F32, MARL_BF16, MARL_F16 or MARL_MXFP4");
    if (num_rows == 0) return MARL_OK;
    if (!d_x || !d_w_codes || !d_w_scales || !d_y) return set_error(MARL_ERR_INVALID, "NULL argument to marl_mx_linear");
    if ((x_type == MARL_MXFP4) != (d_x_scales != nullptr) || (y_type == MARL_MXFP4) != (d_y_scales != nullptr))
        return set_error(MARL_ERR_INVALID, "d_x_scales / d_y_scales belong to MARL_MXFP4 operands, and only to them");
    if (x_type == MARL_MXFP4 ? row_stride != 0 : row_stride != 0 && row_stride < num_cols)
        return set_error(MARL_ERR_INVALID, "row_stride is smaller than num_cols (0 with MARL_MXFP4 rows, which are packed)");
    const size_t xa = x_type == MARL_MXFP4 ? 16 : lb_type_bytes(x_type), ya = y_type == MARL_MXFP4 ? 16 : lb_type_bytes(y_type);
    if (((uintptr_t)d_x & (xa - 1)) != 0 || ((uintptr_t)d_y & (ya - 1)) != 0 || ((uintptr_t)d_w_codes & 15u) != 0 ||
        ((uintptr_t)d_bias & 3u) != 0 || ((uintptr_t)d_workspace & 15u) != 0)
        return set_error(MARL_ERR_INVALID, "codes and the workspace must be 16-byte aligned, the others aligned to their elements");
    if (too_many_blocks(num_rows, num_cols) || too_many_blocks(num_rows, num_out) || num_out > (1 << 22))
        return set_error(MARL_ERR_INVALID, "at most 2^30 - 64 blocks of 32 values on either side and at most 2^22 output features in one call");
    if (!mx_short_rows(num_cols) && num_rows > (int64_t)65535 * 64)
        return set_error(MARL_ERR_INVALID, "of rows of fewer than 8 or more than 512 values at most 4,194,240 in one call");
    if (marl_mx_linear_workspace_bytes(x_type, num_rows, num_cols, num_out) != 0 && !d_workspace)
        return set_error(MARL_ERR_INVALID, "this size needs d_workspace (marl_mx_linear_workspace_bytes bytes)");
    MxLinear P;
    P.x = d_x; P.x_scales = d_x_scales;
    P.rows = num_rows; P.pitch = row_stride ? row_stride : num_cols;
    P.cols = num_cols; P.blocks = (int)lb_blocks(num_cols);
    P.w = d_w_codes; P.w_scales = d_w_scales; P.out = num_out;
    P.bias = d_bias; P.relu = relu != 0;
    P.y = d_y; P.y_scales = d_y_scales;
    P.part = nullptr; P.splits = 1;
    return hip_result(launch_linear(P, x_type, y_type, static_cast<uint8_t*>(d_workspace), reinterpret_cast<hipStream_t>(stream)),
                      "MXFP4 linear launch");
}
