// Activations kept in 8 bits between the forward and the backward pass of the policy's update, for gfx950.
//
//   block of 32 values x along a row, scale 2^e, e the smallest with round(max|x| / 2^e) <= 127 (255 where no value is
//   negative, as behind a ReLU), at least -126 and small enough that 127 (255) of them are finite;
//   code = round(x / 2^e) + 128 (+ 0), ties to even, cut at 127 (255);  scale byte e + 127, 255 for a
//   block that holds an infinity or a NaN, which then reads as NaN throughout.
//   In the non-negative form a positive value never gets code 0, so "code > 0" is the ReLU's own mask, exactly.
//
// Why this form: a code times a power of two is exactly a bfloat16 (eight significant bits), so the weight gradient
// takes the kept activation into the bf16 matrix cores as it stands, and whole numbers up to 127 (the observations) are
// kept exactly.
#include "lowbit.h"

namespace oc {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// scale byte of a block from the bits of its largest |x|: the exponent after adding what takes a mantissa of
// 127.5/64 (255.5/128) or more over to the next power; at float32's largest exponent there is none, and the codes are cut
template <bool POSITIVE>
__device__ __forceinline__ uint32_t act_scale_byte(uint32_t top) {
    if (top >= 0x7F800000u) return 255u;
    const uint32_t e = min((top + (POSITIVE ? 0x8000u : 0x10000u)) >> 23, 254u), off = POSITIVE ? 7u : 6u;
    return e > off ? e - off : 1u;
}

// Four lanes per block, eight values each.  Bound by memory.
template <int TYPE, bool POSITIVE>
__global__ void __launch_bounds__(256)
act_compress_kernel(const void* __restrict__ x, int64_t rows, int cols, int64_t pitch, int blocks,
                    uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    int64_t row;
    int b, quarter;
    split_block(blockIdx.x * 256 + threadIdx.x, (uint32_t)blocks, row, b, quarter);
    if (row >= rows) return;  // whole quads leave together
    float v[8];
    const int64_t at = (int64_t)b * LB_BLOCK + quarter * 8;
    load_eight<TYPE>(x, row * pitch + at, row * pitch + cols, v);
    if (POSITIVE) {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = v[k] < 0.0f ? 0.0f : v[k];  // a NaN stays
    }
    const uint32_t byte = act_scale_byte<POSITIVE>(quad_max(abs_top(v)));
    const float inv = bits_f((254u - min(byte, 253u)) << 23);
    uint32_t c[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        if (POSITIVE) {
            const uint32_t q = (uint32_t)fminf(rintf(v[k] * inv), 255.0f);
            c[k] = v[k] == 0.0f ? 0u : byte == 255u ? 255u : max(q, 1u);
        } else {
            c[k] = byte == 255u ? 128u : (uint32_t)((int)__builtin_amdgcn_fmed3f(rintf(v[k] * inv), -127.0f, 127.0f) + 128);
        }
    }
    uint8_t* out = codes + row * cols + at;
    if (at + 8 <= cols) {
        *reinterpret_cast<u32x2_a1*>(out) = u32x2{c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24, c[4] | c[5] << 8 | c[6] << 16 | c[7] << 24};
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (at + k < cols) out[k] = (uint8_t)c[k];
    }
    if (quarter == 0) scales[row * blocks + b] = (uint8_t)byte;
}

template <int TYPE>
__global__ void __launch_bounds__(256)
act_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t rows, int cols,
                      int blocks, float zero, void* __restrict__ out) {
    int64_t row;
    int b, quarter;
    split_block(blockIdx.x * 256 + threadIdx.x, (uint32_t)blocks, row, b, quarter);
    if (row >= rows) return;
    const int64_t at = (int64_t)b * LB_BLOCK + quarter * 8;
    const float s = scale_value(scales[row * blocks + b]);
    const uint8_t* c = codes + row * cols + at;
    float v[8];
    if (at + 8 <= cols) {
        const u32x2 u = *reinterpret_cast<const u32x2_a1*>(c);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = ((float)((u[k >> 2] >> (8 * (k & 3))) & 255u) - zero) * s;
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = at + k < cols ? ((float)c[k] - zero) * s : 0.0f;
    }
    store_eight<TYPE>(out, row * cols + at, row * cols + cols, v);
}

// ------------------------------------------------------------------------------------------------- weight gradient
//
//   g[m][o]  = grad[m][o], cut to 0 where the layer's kept output has code 0
//   gw[o][i] = sum_m g[m][o] x[m][i],   gb[o] = sum_m g[m][o]
//
// The sum runs over the rows, 32 of them a step of v_mfma_f32_16x16x32_bf16.  x is a bfloat16 exactly.  A float32 g is
// the sum of three bfloat16 numbers exactly (its 24 bits cut into eights), so three products with float32 sums give
// float32's accuracy; a float16 g needs two and a bfloat16 g one.
// Both operands are wanted with the rows innermost: a thread takes 8 rows of two (g) or four (x) columns, and writes 16
// bytes per column and part to LDS, which is the transposition.

struct ActGrad {
    const void* grad;            // [rows][out]
    const uint8_t* mask;         // [rows][out] codes of the kept output, or NULL
    int64_t rows;
    int out, cols, blocks;
    const uint8_t* codes;        // [rows][cols]
    const uint8_t* scales;       // [rows][blocks]
    float zero;                  // 128 or 0
    void* masked;                // [rows][out], written if mask
    float* gw;                   // [splits][out][cols] (the result itself if splits is 1)
    float* gb;                   // [splits][out]
    int splits;
    int64_t per;                 // rows of a split, a multiple of 32
};

template <int TYPE> constexpr int grad_parts() { return TYPE == MARL_F32 ? 3 : TYPE == MARL_F16 ? 2 : 1; }

constexpr int WG_STEP = 32;                 // rows a step
constexpr int WG_PITCH = WG_STEP * 2 + 16;  // LDS bytes per column: the 16 spread columns over the banks

__device__ __forceinline__ uint32_t high_halves(float a, float b) {  // a's upper 16 bits below b's
    return __builtin_amdgcn_perm(f_bits(b), f_bits(a), 0x07060302u);
}

template <int TYPE>
__device__ __forceinline__ void load_two(const void* p, int64_t at, bool two, float& a, float& b) {
    if constexpr (TYPE == MARL_F32) {
        typedef f32x2 f32x2_a4 __attribute__((aligned(4)));
        if (two) {
            const f32x2 v = *reinterpret_cast<const f32x2_a4*>(static_cast<const float*>(p) + at);
            a = v.x; b = v.y;
        } else {
            a = static_cast<const float*>(p)[at]; b = 0.0f;
        }
    } else {
        a = load_one<TYPE>(p, at);
        b = two ? load_one<TYPE>(p, at + 1) : 0.0f;
    }
}

template <int TYPE>
__device__ __forceinline__ void store_two(void* p, int64_t at, bool two, float a, float b) {
    if constexpr (TYPE == MARL_F32) {
        static_cast<float*>(p)[at] = a;
        if (two) static_cast<float*>(p)[at + 1] = b;
    } else {
        static_cast<uint16_t*>(p)[at] = to_half_type<TYPE>(a);
        if (two) static_cast<uint16_t*>(p)[at + 1] = to_half_type<TYPE>(b);
    }
}

// A workgroup of four waves has BO output features and BI input features, each wave BO/WO by BI/WI of them.
template <int TYPE, int BO, int BI, int WO, int WI>
__global__ void __launch_bounds__(256)
act_weight_grad_kernel(ActGrad P) {
    static_assert(WO * WI == 4, "four waves");
    constexpr int PARTS = grad_parts<TYPE>();
    constexpr int TO = BO / WO / 16, TI = BI / WI / 16;
    __shared__ __align__(16) uint8_t A[PARTS][BO][WG_PITCH];
    __shared__ __align__(16) uint8_t B[BI][WG_PITCH];
    __shared__ float bias_sum[BO][4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 15, g = lane >> 4;
    const int o0 = blockIdx.y * BO, i0 = blockIdx.x * BI;
    const int wo = (wave / WI) * (BO / WO), wi = (wave % WI) * (BI / WI);
    const int64_t first = (int64_t)blockIdx.z * P.per, last = min(P.rows, first + P.per);
    const bool leader = blockIdx.x == 0;  // also writes the cut gradient and sums it

    constexpr int GITEMS = BO * 2, XITEMS = BI;  // (group of 8 rows, 2 columns), (group of 8 rows, 4 columns)
    constexpr int GN = (GITEMS + 255) / 256, XN = (XITEMS + 255) / 256;
    float bsum[GN][2];
#pragma unroll
    for (int q = 0; q < GN; ++q) bsum[q][0] = bsum[q][1] = 0.0f;
    f32x4 acc[TO][TI];
#pragma unroll
    for (int a = 0; a < TO; ++a)
#pragma unroll
        for (int b = 0; b < TI; ++b) acc[a][b] = f32x4{0, 0, 0, 0};

    for (int64_t m0 = first; m0 < last; m0 += WG_STEP) {
#pragma unroll
        for (int q = 0; q < GN; ++q) {
            const int it = tid + q * 256;
            if (GITEMS % 256 != 0 && it >= GITEMS) break;
            const int pair = it % (BO / 2), mg = it / (BO / 2), o = o0 + 2 * pair;
            float a[8], b[8];
            uint32_t top = 0;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int64_t m = m0 + mg * 8 + k;
                a[k] = b[k] = 0.0f;
                if (m < last && o < P.out) {
                    const bool two = o + 1 < P.out;
                    load_two<TYPE>(P.grad, m * P.out + o, two, a[k], b[k]);
                    if (P.mask) {
                        a[k] = P.mask[m * P.out + o] ? a[k] : 0.0f;
                        b[k] = two && P.mask[m * P.out + o + 1] ? b[k] : 0.0f;
                        if (leader) store_two<TYPE>(P.masked, m * P.out + o, two, a[k], b[k]);
                    }
                }
                top = max(top, max(f_bits(a[k]) & 0x7FFFFFFFu, f_bits(b[k]) & 0x7FFFFFFFu));
            }
            bsum[q][0] += ((a[0] + a[1]) + (a[2] + a[3])) + ((a[4] + a[5]) + (a[6] + a[7]));
            bsum[q][1] += ((b[0] + b[1]) + (b[2] + b[3])) + ((b[4] + b[5]) + (b[6] + b[7]));
            const bool wild = top >= 0x7F800000u;  // an infinity minus itself is no number: it has no lower parts
#pragma unroll
            for (int p = 0; p < PARTS; ++p) {
                u32x4 ua, ub;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    ua[k] = high_halves(a[2 * k], a[2 * k + 1]);
                    ub[k] = high_halves(b[2 * k], b[2 * k + 1]);
                }
                *reinterpret_cast<u32x4*>(&A[p][2 * pair][mg * 16]) = ua;
                *reinterpret_cast<u32x4*>(&A[p][2 * pair + 1][mg * 16]) = ub;
                if (p + 1 < PARTS) {
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        a[k] = wild && isinf(a[k]) ? 0.0f : a[k] - bits_f(f_bits(a[k]) & 0xFFFF0000u);
                        b[k] = wild && isinf(b[k]) ? 0.0f : b[k] - bits_f(f_bits(b[k]) & 0xFFFF0000u);
                    }
                }
            }
        }
#pragma unroll
        for (int q = 0; q < XN; ++q) {
            const int it = tid + q * 256;
            if (XITEMS % 256 != 0 && it >= XITEMS) break;
            const int four = it % (BI / 4), mg = it / (BI / 4), i = i0 + 4 * four;
            float v[4][8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int64_t m = m0 + mg * 8 + k;
#pragma unroll
                for (int c = 0; c < 4; ++c) v[c][k] = 0.0f;
                if (m < last && i < P.cols) {
                    const uint8_t* at = P.codes + m * P.cols + i;
                    const float s = scale_value(P.scales[m * P.blocks + i / LB_BLOCK]);
                    uint32_t u;
                    if (i + 4 <= P.cols) u = *reinterpret_cast<const u32_a1*>(at);
                    else {
                        u = at[0];
                        if (i + 1 < P.cols) u |= (uint32_t)at[1] << 8;
                        if (i + 2 < P.cols) u |= (uint32_t)at[2] << 16;
                    }
#pragma unroll
                    for (int c = 0; c < 4; ++c) v[c][k] = ((float)((u >> (8 * c)) & 255u) - P.zero) * s;
                }
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                u32x4 u;
#pragma unroll
                for (int k = 0; k < 4; ++k) u[k] = high_halves(v[c][2 * k], v[c][2 * k + 1]);
                *reinterpret_cast<u32x4*>(&B[4 * four + c][mg * 16]) = u;
            }
        }
        __syncthreads();
        bf16x8 x[TI];
#pragma unroll
        for (int b = 0; b < TI; ++b) x[b] = *reinterpret_cast<const bf16x8*>(&B[wi + b * 16 + r][g * 16]);
#pragma unroll
        for (int p = PARTS - 1; p >= 0; --p)
#pragma unroll
            for (int a = 0; a < TO; ++a) {
                const bf16x8 y = *reinterpret_cast<const bf16x8*>(&A[p][wo + a * 16 + r][g * 16]);
#pragma unroll
                for (int b = 0; b < TI; ++b) acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(y, x[b], acc[a][b], 0, 0, 0);
            }
        __syncthreads();
    }

    float* gw = P.gw + (size_t)blockIdx.z * P.out * P.cols;
#pragma unroll
    for (int a = 0; a < TO; ++a)
#pragma unroll
        for (int b = 0; b < TI; ++b)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int o = o0 + wo + a * 16 + g * 4 + k, i = i0 + wi + b * 16 + r;
                if (o < P.out && i < P.cols) gw[(size_t)o * P.cols + i] = acc[a][b][k];
            }
    if (leader) {
#pragma unroll
        for (int q = 0; q < GN; ++q) {
            const int it = tid + q * 256;
            if (GITEMS % 256 != 0 && it >= GITEMS) break;
            const int pair = it % (BO / 2), mg = it / (BO / 2);
            bias_sum[2 * pair][mg] = bsum[q][0];
            bias_sum[2 * pair + 1][mg] = bsum[q][1];
        }
        __syncthreads();
        for (int o = tid; o < BO; o += 256)
            if (o0 + o < P.out)
                P.gb[(size_t)blockIdx.z * P.out + o0 + o] = (bias_sum[o][0] + bias_sum[o][1]) + (bias_sum[o][2] + bias_sum[o][3]);
    }
}

// Sums of the splits in their order, in double (hundreds of them, one after the other): the weight's entries, then the
// bias's
__global__ void __launch_bounds__(256)
act_join_kernel(const float* __restrict__ part_w, const float* __restrict__ part_b, int64_t nw, int nb, int splits,
                float* __restrict__ gw, float* __restrict__ gb) {
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const bool bias = at >= nw;
    if (at >= nw + nb) return;
    const float* p = bias ? part_b + (at - nw) : part_w + at;
    const int64_t step = bias ? nb : nw;
    double s = 0.0;
    for (int k = 0; k < splits; ++k) s += (double)p[k * step];
    if (bias) gb[at - nw] = (float)s;
    else gw[at] = (float)s;
}

// ------------------------------------------------------------------------------------------------------------ host

struct ActCut { int bo, bi, splits; int64_t per; };
static ActCut act_cut(int64_t rows, int out, int cols) {
    ActCut c;
    c.bo = out <= 16 ? 16 : 64;
    c.bi = out <= 16 ? 256 : 64;
    const int64_t tiles = (int64_t)((out + c.bo - 1) / c.bo) * ((cols + c.bi - 1) / c.bi);
    const int64_t steps = (rows + WG_STEP - 1) / WG_STEP;
    int64_t s = 1024 / tiles;
    s = s < 1 ? 1 : s;
    const int64_t most = (steps + 3) / 4;  // at least four steps each
    s = s > most ? most : s;
    const int64_t each = (steps + s - 1) / s;
    c.per = each * WG_STEP;
    c.splits = (int)((steps + each - 1) / each);
    return c;
}

template <int TYPE>
static void launch_weight_grad_type(const ActGrad& P, const ActCut& c, dim3 grid, hipStream_t stream) {
    if (c.bo == 16) hipLaunchKernelGGL((act_weight_grad_kernel<TYPE, 16, 256, 1, 4>), grid, dim3(256), 0, stream, P);
    else hipLaunchKernelGGL((act_weight_grad_kernel<TYPE, 64, 64, 2, 2>), grid, dim3(256), 0, stream, P);
}

static int act_hip(hipError_t e, const char* what) {
    if (e == hipSuccess) return MARL_OK;
    return set_error(MARL_ERR_HIP, std::string(what) + ": " + hipGetErrorString(e));
}

}  // namespace oc

using namespace oc;

extern "C" int marl_act_compress(const void* d_x, int x_type, int64_t num_rows, int num_cols, int64_t row_stride, int nonnegative,
                                 uint8_t* d_codes, uint8_t* d_scales, void* stream) {
    if (num_rows < 0 || num_cols <= 0) return set_error(MARL_ERR_INVALID, "num_rows must not be negative and num_cols must be positive");
    if (x_type != MARL_F32 && x_type != MARL_BF16 && x_type != MARL_F16)
        return set_error(MARL_ERR_INVALID, "x_type must be MARL_F32, MARL_BF16 or MARL_F16");
    if (num_rows == 0) return MARL_OK;
    if (!d_x || !d_codes || !d_scales) return set_error(MARL_ERR_INVALID, "NULL argument to marl_act_compress");
    if (row_stride == 0) row_stride = num_cols;
    if (row_stride < num_cols) return set_error(MARL_ERR_INVALID, "row_stride is smaller than num_cols");
    if (((uintptr_t)d_x & (lb_type_bytes(x_type) - 1)) != 0) return set_error(MARL_ERR_INVALID, "d_x must be aligned to its elements");
    if (too_many_blocks(num_rows, num_cols)) return set_error(MARL_ERR_INVALID, "2^30 or more blocks of 32 values in one call");
    const int blocks = (int)lb_blocks(num_cols);
    auto pick = [&](auto positive) {
        constexpr bool pos = decltype(positive)::value;
        return x_type == MARL_F32 ? act_compress_kernel<MARL_F32, pos> : x_type == MARL_BF16 ? act_compress_kernel<MARL_BF16, pos>
                                                                                             : act_compress_kernel<MARL_F16, pos>;
    };
    auto kernel = nonnegative ? pick(std::true_type{}) : pick(std::false_type{});
    hipLaunchKernelGGL(kernel, dim3(block_grid(num_rows, num_cols)), dim3(256), 0, reinterpret_cast<hipStream_t>(stream), d_x, num_rows,
                       num_cols, row_stride, blocks, d_codes, d_scales);
    return act_hip(hipGetLastError(), "activation compression launch");
}

extern "C" int marl_act_dequantize(const uint8_t* d_codes, const uint8_t* d_scales, int64_t num_rows, int num_cols, int nonnegative,
                                   int out_type, void* d_out, void* stream) {
    if (num_rows < 0 || num_cols <= 0) return set_error(MARL_ERR_INVALID, "num_rows must not be negative and num_cols must be positive");
    if (out_type != MARL_F32 && out_type != MARL_BF16 && out_type != MARL_F16)
        return set_error(MARL_ERR_INVALID, "out_type must be MARL_F32, MARL_BF16 or MARL_F16");
    if (num_rows == 0) return MARL_OK;
    if (!d_codes || !d_scales || !d_out) return set_error(MARL_ERR_INVALID, "NULL argument to marl_act_dequantize");
    if (((uintptr_t)d_out & (lb_type_bytes(out_type) - 1)) != 0) return set_error(MARL_ERR_INVALID, "d_out must be aligned to its elements");
    if (too_many_blocks(num_rows, num_cols)) return set_error(MARL_ERR_INVALID, "2^30 or more blocks of 32 values in one call");
    auto kernel = out_type == MARL_F32 ? act_dequantize_kernel<MARL_F32> : out_type == MARL_BF16 ? act_dequantize_kernel<MARL_BF16>
                                                                                                 : act_dequantize_kernel<MARL_F16>;
    hipLaunchKernelGGL(kernel, dim3(block_grid(num_rows, num_cols)), dim3(256), 0, reinterpret_cast<hipStream_t>(stream), d_codes, d_scales,
                       num_rows, num_cols, (int)lb_blocks(num_cols), nonnegative ? 0.0f : 128.0f, d_out);
    return act_hip(hipGetLastError(), "activation read-back launch");
}

extern "C" size_t marl_act_weight_grad_workspace_bytes(int64_t num_rows, int num_out, int num_cols) {
    if (num_rows <= 0 || num_out <= 0 || num_cols <= 0) return 0;
    const ActCut c = act_cut(num_rows, num_out, num_cols);
    return c.splits == 1 ? 0 : (size_t)c.splits * ((size_t)num_out * num_cols + num_out) * sizeof(float);
}

extern "C" int marl_act_weight_grad(const void* d_grad, int grad_type, int64_t num_rows, int num_out, const uint8_t* d_codes,
                                    const uint8_t* d_scales, int num_cols, int nonnegative, const uint8_t* d_mask_codes,
                                    void* d_masked_grad, float* d_grad_weight, float* d_grad_bias, void* d_workspace, void* stream) {
    if (num_rows <= 0 || num_out <= 0 || num_cols <= 0)
        return set_error(MARL_ERR_INVALID, "num_rows, num_out and num_cols must be positive");
    if (grad_type != MARL_F32 && grad_type != MARL_BF16 && grad_type != MARL_F16)
        return set_error(MARL_ERR_INVALID, "grad_type must be MARL_F32, MARL_BF16 or MARL_F16");
    if (!d_grad || !d_codes || !d_scales || !d_grad_weight || !d_grad_bias)
        return set_error(MARL_ERR_INVALID, "NULL argument to marl_act_weight_grad");
    if ((d_mask_codes == nullptr) != (d_masked_grad == nullptr))
        return set_error(MARL_ERR_INVALID, "d_mask_codes and d_masked_grad go together");
    if (d_masked_grad == d_grad) return set_error(MARL_ERR_INVALID, "d_masked_grad must not be d_grad");
    const size_t ga = lb_type_bytes(grad_type) - 1;
    if (((uintptr_t)d_grad & ga) != 0 || ((uintptr_t)d_masked_grad & ga) != 0 || ((uintptr_t)d_grad_weight & 3u) != 0 ||
        ((uintptr_t)d_grad_bias & 3u) != 0 || ((uintptr_t)d_workspace & 15u) != 0)
        return set_error(MARL_ERR_INVALID, "d_workspace must be 16-byte aligned, the others aligned to their elements");
    if (num_rows >= ((int64_t)1 << 40) || num_out > (1 << 20) || num_cols > (1 << 20) || (int64_t)num_out * num_cols > ((int64_t)1 << 31))
        return set_error(MARL_ERR_INVALID, "at most 2^40 rows, 2^20 features on a side and 2^31 weights");
    const ActCut c = act_cut(num_rows, num_out, num_cols);
    if (c.splits > 1 && !d_workspace)
        return set_error(MARL_ERR_INVALID, "this size needs d_workspace (marl_act_weight_grad_workspace_bytes bytes)");
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const int64_t nw = (int64_t)num_out * num_cols;
    ActGrad P;
    P.grad = d_grad; P.mask = d_mask_codes; P.rows = num_rows; P.out = num_out; P.cols = num_cols;
    P.blocks = (int)lb_blocks(num_cols);
    P.codes = d_codes; P.scales = d_scales; P.zero = nonnegative ? 0.0f : 128.0f; P.masked = d_masked_grad;
    P.splits = c.splits; P.per = c.per;
    P.gw = c.splits == 1 ? d_grad_weight : static_cast<float*>(d_workspace);
    P.gb = c.splits == 1 ? d_grad_bias : static_cast<float*>(d_workspace) + c.splits * nw;
    const dim3 grid((num_cols + c.bi - 1) / c.bi, (num_out + c.bo - 1) / c.bo, c.splits);
    if (grad_type == MARL_F32) launch_weight_grad_type<MARL_F32>(P, c, grid, s);
    else if (grad_type == MARL_BF16) launch_weight_grad_type<MARL_BF16>(P, c, grid, s);
    else launch_weight_grad_type<MARL_F16>(P, c, grid, s);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || c.splits == 1) return act_hip(e, "weight gradient launch");
    const int64_t threads = nw + num_out;
    hipLaunchKernelGGL(act_join_kernel, dim3((uint32_t)((threads + 255) / 256)), dim3(256), 0, s, P.gw, P.gb, nw, num_out, c.splits,
                       d_grad_weight, d_grad_bias);
    return act_hip(hipGetLastError(), "weight gradient join launch");
}
