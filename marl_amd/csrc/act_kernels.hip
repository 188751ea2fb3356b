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

// Four lanes per block, eight values each.  Bound by memory: 131072 x 512 float32 values are compressed and read back in 108
// us, 686 MB, of which the codes between the two stay in the last-level cache.  (Two or four items a thread, their loads
// together, are slower: 58, 61 and 64 us for compressing.)
template <int TYPE, bool POSITIVE, bool NT>
__global__ void __launch_bounds__(256)
act_compress_kernel(const void* __restrict__ x, int64_t rows, int cols, int64_t pitch, int blocks,
                    uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    int64_t row;
    int b, quarter;
    split_block(blockIdx.x * 256 + threadIdx.x, (uint32_t)blocks, row, b, quarter);
    if (row >= rows) return;  // whole quads leave together
    float v[8];
    const int64_t at = (int64_t)b * LB_BLOCK + quarter * 8;
    load_eight<TYPE, NT>(x, row * pitch + at, row * pitch + cols, v);
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
// the sum of three bfloat16 numbers exactly (its 24 bits cut into eights; of a g below 2^-109 what lies under bfloat16's
// smallest, 2^-133, is lost), so three products with float32 sums give float32's accuracy; a float16 g needs two and a
// bfloat16 g one.
// Both operands are wanted with the rows innermost: a thread takes 4 (g) or 8 rows (x) of four columns and writes 8 or 16
// bytes per column and part to LDS, which is the transposition.

struct ActGrad {
    const void* grad;            // [rows][out]
    const uint8_t* mask;         // [rows][out] codes of the kept output, or NULL
    int64_t rows;
    int out, cols, blocks;
    const uint8_t* codes;        // [rows][cols]
    const uint8_t* scales;       // [rows][blocks]
    float zero;                  // 128 or 0
    void* masked;                // [rows][out], or NULL: a mask whose cut gradient nothing reads
    float* gw;                   // [splits][out][cols] (the result itself if splits is 1)
    float* gb;                   // [splits][out]
    int splits;
};

// What is done about the mask: there is none; the gradient is cut; it is cut and written.  (The last two as one kernel that asks
// whether there is a place to write to: 128 us instead of 124 at 131072 x 256 x 512 in float32.  Not written: 119.)
enum { UNCUT, CUT, CUT_KEPT };

template <int TYPE> constexpr int grad_parts() { return TYPE == MARL_F32 ? 3 : TYPE == MARL_F16 ? 2 : 1; }

constexpr int WG_STEP = 32;                 // rows a step
constexpr int WG_PITCH = WG_STEP * 2;       // LDS bytes per column, four pieces of 8 rows

// Where the piece of rows 8 p .. 8 p + 7 of a column lies within it: turned by the column's place, so that the 16 columns
// that a fragment's lanes read lie in different banks (4.2 cycles a read of a wave; 8.0 without, or with padded columns).
__device__ __forceinline__ int piece(int place, int p) { return (p ^ (place >> 1 & 3)) * 16; }

__device__ __forceinline__ uint32_t high_halves(float a, float b) {  // a's upper 16 bits below b's
    return __builtin_amdgcn_perm(f_bits(b), f_bits(a), 0x07060302u);
}

// Four neighbouring values of a row as they come from memory (16-bit types: two words).  The last group of a row that is no
// multiple of four is the row's last four values, moved down by `back` places when they are used: what then stands behind
// the row's end does not matter, and memory behind it is not touched.  Where one of the operands has rows of fewer than four values, all are read one by one.
template <int TYPE, bool NARROW>
__device__ __forceinline__ u32x4 load_four(const void* p, uint32_t at, int have) {
    if constexpr (NARROW) {
        u32x4 u = {0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < 4; ++k) u[k] = f_bits(load_one<TYPE>(p, at + min(k, have - 1)));
        return u;
    }
    if constexpr (TYPE == MARL_F32) {
        typedef u32x4 u32x4_a4 __attribute__((aligned(4)));
        return *reinterpret_cast<const u32x4_a4*>(static_cast<const uint8_t*>(p) + at * 4u);
    } else {
        typedef u32x2 u32x2_a2 __attribute__((aligned(2)));
        const u32x2 q = *reinterpret_cast<const u32x2_a2*>(static_cast<const uint8_t*>(p) + at * 2u);
        return u32x4{q.x, q.y, 0, 0};
    }
}
template <int TYPE, bool NARROW>
__device__ __forceinline__ void use_four(u32x4 q, int back, float (&v)[4]) {
    float a, b, c, d;
    if constexpr (TYPE == MARL_F32 || NARROW) {
        a = bits_f(q.x); b = bits_f(q.y); c = bits_f(q.z); d = bits_f(q.w);
    } else if constexpr (TYPE == MARL_BF16) {
        a = bits_f(q.x << 16); b = bits_f(q.x & 0xFFFF0000u); c = bits_f(q.y << 16); d = bits_f(q.y & 0xFFFF0000u);
    } else {
        a = half_lo(q.x); b = half_hi(q.x); c = half_lo(q.y); d = half_hi(q.y);
    }
    if (back) {
        a = back == 1 ? b : back == 2 ? c : d;
        b = back == 1 ? c : d;
        c = d;
    }
    v[0] = a; v[1] = b; v[2] = c; v[3] = d;
}
template <bool NARROW>
__device__ __forceinline__ uint32_t load_four_bytes(const uint8_t* p, uint32_t at, int have) {
    if constexpr (NARROW) {
        uint32_t u = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) u |= (uint32_t)p[at + min(k, have - 1)] << (8 * k);
        return u;
    }
    return *reinterpret_cast<const u32_a1*>(p + at);
}

// A workgroup has BO output features and BI input features, its waves (WO x WI of them) BO/WO by 64 each.  LDS holds two
// steps: while the waves multiply one, they convert the next, whose loads went out two steps earlier; one barrier a step.
// Some waves convert x and the others g, the latter before they multiply and the former after it, so that on each SIMD
// the matrix unit and the vector unit have work at the same time.
// A column of the tile lies in LDS at (column % 4) * (columns / 4) + column / 4, so that the lanes of a wave, which take
// four neighbouring columns each, write to neighbouring places, and a lane's results are four neighbouring inputs.
//
// 131072 rows x 256 outputs x 512 inputs, float32 gradient with a mask that is written: 117 us and 6 us for the joining kernel (float16, two
// products, 108; bfloat16, one, 89, without a mask 69).  The float32 form has 256 registers and 12 bytes of scratch a thread; without
// the written gradient it has none, and takes 119 us instead of 137 at 131072 x 512 x 202.  237 MB come from HBM once and 168 MB go there, 78 us at a copy's rate; three bf16 products take 85 us at
// the rate of a large library product, 41 us at the matrix units' own.  Those are busy 37 % of the time and the vector units as
// long; g and x reach the compute units twice, 470 MB at 4.1 TB/s, which is what loads alone in this order reach (4.5).
// Measured and no faster, 118 to 137 us: 1024 threads; waves that only load and convert before waves that only multiply, over
// three buffers; loads three and four steps ahead; a quarter fewer vector instructions; fewer output features to the waves that
// convert g.  Two workgroups a compute unit double the partial sums (34 MB): 10 us more.
// Not tried: 128 x 512, which would read g and its mask once and x twice (306 MB instead of 470).
template <int TYPE, int BO, int BI, int WO, int WI, int MASK, bool NARROW>
struct WeightGrad {
    static constexpr int PARTS = grad_parts<TYPE>(), BYTES = TYPE == MARL_F32 ? 4 : 2;
    static constexpr int THREADS = 64 * WO * WI, TO = BO / WO / 16, GITEMS = 2 * BO, XITEMS = BI;
    static_assert(BI == 64 * WI && GITEMS <= THREADS && XITEMS <= THREADS, "a wave has 64 input features, a thread one item of each kind");

    static constexpr bool STEADY = BO == 128;  // every step makes the same loads

    struct Lds {
        uint8_t A[2][PARTS][BO][WG_PITCH];
        uint8_t B[2][BI][WG_PITCH];
    };
    struct RawX { uint32_t x[8], s[2]; };  // 8 rows of 4 columns and two of the rows' scales
    struct RawG { u32x4 g[4]; uint32_t m[4]; };  // 4 rows of 4 columns

    const ActGrad& P;
    Lds& S;
    int64_t first, stride, last;
    int o0, i0, lane, wo, wi;
    bool leader;  // also writes the cut gradient and sums it
    int xc, xr, xi, xback, xhave, gc, gr, go, gback, ghave;
    bool has_g;
    float bsum[4] = {0, 0, 0, 0};
    f32x4 acc[TO][4];

    // Rows behind the last are the last one again (their g counts as 0), and in the largest tile, which has many steps, so are
    // steps behind the last: were the loads left out on some path, the compiler would no longer know how many are under way, and
    // wait for all (131072 x 512 x 202 with a mask: 100 us in bfloat16, 143 in float32; so 130 and 148).  In the others the steps
    // there are to spare cost more than that (65000 x 8 x 256 in bfloat16: 14.4 us, with them 15.5).  A step's place is the same
    // for the whole workgroup, what differs from thread to thread is a 32-bit offset (at most 32 rows of 2^20 values).
    template <bool X, bool G>
    __device__ __forceinline__ void fetch(RawX& x, RawG& g, int64_t m0) const {
        if (!STEADY && m0 >= last) return;
        m0 = min(m0, last - 1);
        const int lim = (int)min(last - 1 - m0, (int64_t)WG_STEP - 1);
        if constexpr (X) {
            const uint8_t* codes = P.codes + m0 * P.cols;
            const uint8_t* scales = P.scales + m0 * P.blocks;
#pragma unroll
            for (int k = 0; k < 8; ++k) x.x[k] = load_four_bytes<NARROW>(codes, __umul24(min(xr + k, lim), P.cols) + (xi - xback), xhave);
            // a quad's four lanes have the same block of 32: each takes the scales of two of the eight rows
#pragma unroll
            for (int k = 0; k < 2; ++k) x.s[k] = scales[__umul24(min(xr + 4 * k + (lane & 3), lim), P.blocks) + xi / LB_BLOCK];
        }
        if constexpr (G) {
            const uint8_t* grad = static_cast<const uint8_t*>(P.grad) + m0 * P.out * BYTES;
            const uint8_t* mask = MASK ? P.mask + m0 * P.out : nullptr;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t at = __umul24(min(gr + k, lim), P.out) + (go - gback);
                g.g[k] = load_four<TYPE, NARROW>(grad, at, ghave);
                if constexpr (MASK) g.m[k] = load_four_bytes<NARROW>(mask, at, ghave);
            }
        }
    }

    __device__ __forceinline__ void convert_x(const RawX& raw, int buf) const {
        float s[8];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int v = (int)f_bits(scale_value(raw.s[k]));
            s[4 * k] = bits_f(__builtin_amdgcn_update_dpp(0, v, 0x00, 0xF, 0xF, true));  // quad_perm: lane 0's
            s[4 * k + 1] = bits_f(__builtin_amdgcn_update_dpp(0, v, 0x55, 0xF, 0xF, true));
            s[4 * k + 2] = bits_f(__builtin_amdgcn_update_dpp(0, v, 0xAA, 0xF, 0xF, true));
            s[4 * k + 3] = bits_f(__builtin_amdgcn_update_dpp(0, v, 0xFF, 0xF, 0xF, true));
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            u32x4 u;
#pragma unroll
            for (int k = 0; k < 4; ++k) {  // every step of it is exact (128 times the largest scale, taken off afterwards, would not be)
                const uint32_t xa = raw.x[2 * k] >> (8 * xback), xb = raw.x[2 * k + 1] >> (8 * xback);
                u[k] = high_halves(((float)(xa >> (8 * c) & 255u) - P.zero) * s[2 * k], ((float)(xb >> (8 * c) & 255u) - P.zero) * s[2 * k + 1]);
            }
            *reinterpret_cast<u32x4*>(&S.B[buf][c * (BI / 4) + xc][piece(c * (BI / 4) + xc, xr >> 3)]) = u;
        }
    }

    __device__ __forceinline__ void convert_g(const RawG& raw, int64_t m0, int buf) {
        float v[4][4];
        float odd = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            use_four<TYPE, NARROW>(raw.g[k], gback, v[k]);
            const bool there = m0 + gr + k < last;
            const uint32_t m = MASK ? (there ? raw.m[k] >> (8 * gback) : 0u) : there ? 0xFFFFFFFFu : 0u;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                v[k][c] = m & (255u << (8 * c)) ? v[k][c] : 0.0f;
                if (PARTS > 1) odd = fmaf(v[k][c], 0.0f, odd);
            }
        }
        if (leader) {
#pragma unroll
            for (int c = 0; c < 4; ++c) bsum[c] += (v[0][c] + v[1][c]) + (v[2][c] + v[3][c]);
            if (MASK == CUT_KEPT) write_masked(v, m0);
        }
        const bool wild = odd != 0.0f;  // an infinity or a NaN among them
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
#pragma unroll
            for (int c = 0; c < 4; ++c)
                *reinterpret_cast<u32x2*>(&S.A[buf][p][c * (BO / 4) + gc][piece(c * (BO / 4) + gc, gr >> 3) + (gr & 4) * 2]) =
                    u32x2{high_halves(v[0][c], v[1][c]), high_halves(v[2][c], v[3][c])};
            if (p + 1 == PARTS) break;
            if (p == 0 && wild) {  // an infinity minus itself is no number: it has no lower parts
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (int c = 0; c < 4; ++c) v[k][c] = isinf(v[k][c]) ? 0.0f : v[k][c];
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (int c = 0; c < 4; ++c) v[k][c] -= bits_f(f_bits(v[k][c]) & 0xFFFF0000u);
                continue;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int c = 0; c < 4; ++c) v[k][c] -= bits_f(f_bits(v[k][c]) & 0xFFFF0000u);
        }
    }
    __device__ __forceinline__ void write_masked(const float (&v)[4][4], int64_t m0) const {
        const int c0 = o0 + 4 * gc;
        if (c0 >= P.out) return;
        uint8_t* masked = static_cast<uint8_t*>(P.masked) + m0 * P.out * BYTES;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (m0 + gr + k >= last) continue;
            const uint32_t at = (uint32_t)((gr + k) * P.out + c0);
            if (c0 + 4 <= P.out) {
                if constexpr (TYPE == MARL_F32) {
                    *reinterpret_cast<f32x4_a4*>(masked + at * 4u) = f32x4{v[k][0], v[k][1], v[k][2], v[k][3]};
                } else {
                    typedef u32x2 u32x2_a2 __attribute__((aligned(2)));
                    *reinterpret_cast<u32x2_a2*>(masked + at * 2u) =
                        u32x2{(uint32_t)to_half_type<TYPE>(v[k][0]) | (uint32_t)to_half_type<TYPE>(v[k][1]) << 16,
                              (uint32_t)to_half_type<TYPE>(v[k][2]) | (uint32_t)to_half_type<TYPE>(v[k][3]) << 16};
                }
            } else {
#pragma unroll
                for (int c = 0; c < 3; ++c) {
                    if (c0 + c >= P.out) continue;
                    if constexpr (TYPE == MARL_F32) *reinterpret_cast<float*>(masked + (at + c) * 4u) = v[k][c];
                    else *reinterpret_cast<uint16_t*>(masked + (at + c) * 2u) = to_half_type<TYPE>(v[k][c]);
                }
            }
        }
    }

    __device__ __forceinline__ void multiply(int buf) {
        const int r = lane & 15, g = lane >> 4;
        bf16x8 x[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) x[b] = *reinterpret_cast<const bf16x8*>(&S.B[buf][b * (BI / 4) + wi + r][piece(wi + r, g)]);
        // the next 16 output features' fragments are on their way while these multiply, and no more: registers are short
        bf16x8 y[2][PARTS];
#pragma unroll
        for (int p = 0; p < PARTS; ++p) y[0][p] = *reinterpret_cast<const bf16x8*>(&S.A[buf][p][wo + r][piece(r, g)]);
#pragma unroll
        for (int a = 0; a < TO; ++a) {
            if (a + 1 < TO) {
#pragma unroll
                for (int p = 0; p < PARTS; ++p)
                    y[(a + 1) & 1][p] = *reinterpret_cast<const bf16x8*>(&S.A[buf][p][wo + (a + 1) * 16 + r][piece(r, g)]);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int p = PARTS - 1; p >= 0; --p)
#pragma unroll
                for (int b = 0; b < 4; ++b) acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(y[a & 1][p], x[b], acc[a][b], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
    }

    template <bool X, bool G>
    __device__ __forceinline__ void convert(const RawX& x, const RawG& g, int64_t m0, int buf) {
        if (!STEADY && m0 >= last) return;
        if constexpr (X) convert_x(x, buf);
        if constexpr (G)
            if (has_g) convert_g(g, m0, buf);
    }

    template <bool X, bool G>
    __device__ __forceinline__ void step(RawX& x, RawG& g, int64_t m0, int buf) {
        if constexpr (X) multiply(buf);
        convert<X, G>(x, g, m0 + stride, buf ^ 1);
        fetch<X, G>(x, g, m0 + 3 * stride);
        if constexpr (!X) multiply(buf);
        __syncthreads();
    }

    template <bool X, bool G>
    __device__ __forceinline__ void walk() {
        RawX x0, x1;
        RawG g0, g1;
        fetch<X, G>(x0, g0, first);
        fetch<X, G>(x1, g1, first + stride);
        convert<X, G>(x0, g0, first, 0);
        fetch<X, G>(x0, g0, first + 2 * stride);
        __syncthreads();
        for (int64_t m0 = first; m0 < last; m0 += 2 * stride) {
            step<X, G>(x1, g1, m0, 0);
            if (m0 + stride >= last) break;
            step<X, G>(x0, g0, m0 + stride, 1);
        }
    }

    __device__ __forceinline__ void run(int split, int tile) {
        const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        lane = tid & 63;
        const int ti = (P.cols + BI - 1) / BI;
        o0 = tile / ti * BO;
        i0 = tile % ti * BI;
        wo = wave / WI * (BO / WO);
        wi = wave % WI * 16;
        // the splits take turns at the steps: what runs at the same time reads one stretch of memory
        first = (int64_t)split * WG_STEP;
        stride = (int64_t)P.splits * WG_STEP;
        last = P.rows;
        leader = i0 == 0;
        xc = tid % (BI / 4);
        xr = tid / (BI / 4) * 8;
        const int git = tid - (THREADS - GITEMS);  // the last threads have g
        has_g = git >= 0;
        gc = git & (BO / 4 - 1);
        gr = has_g ? git / (BO / 4) * 4 : 0;
        // Columns behind the end: any that exist, their results are not stored.  With fewer than four columns (NARROW) a
        // group is the columns that there are from its first on.
        xi = min(i0 + 4 * xc, P.cols - 1);
        go = min(o0 + 4 * gc, P.out - 1);
        xback = NARROW ? 0 : max(xi + 4 - P.cols, 0);
        gback = NARROW ? 0 : max(go + 4 - P.out, 0);
        xhave = P.cols - xi;
        ghave = P.out - go;
#pragma unroll
        for (int a = 0; a < TO; ++a)
#pragma unroll
            for (int b = 0; b < 4; ++b) acc[a][b] = f32x4{0, 0, 0, 0};

        // what a wave converts; each form passes the same barriers, and only those that the tile has are there
        const bool wave_x = wave * 64 < XITEMS, wave_g = wave * 64 + 63 >= THREADS - GITEMS;
        if constexpr (XITEMS + GITEMS > THREADS) {
            static_assert(XITEMS == THREADS, "where some have both, all have x");
            if (wave_g) walk<true, true>();
            else walk<true, false>();
        } else if (wave_x) {
            walk<true, false>();
        } else if (wave_g) {
            walk<false, true>();
        } else if constexpr (XITEMS + GITEMS < THREADS) {
            walk<false, false>();
        }

        const int r = lane & 15, g = lane >> 4, ic = i0 + 4 * (wi + r);
        float* gw = P.gw + (size_t)split * P.out * P.cols;
#pragma unroll
        for (int a = 0; a < TO; ++a)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int place = wo + a * 16 + g * 4 + k, oc = o0 + 4 * (place & (BO / 4 - 1)) + place / (BO / 4);
                if (oc >= P.out) continue;
                float* to = gw + (size_t)oc * P.cols + ic;
                if (ic + 4 <= P.cols) {
                    *reinterpret_cast<f32x4_a4*>(to) = f32x4{acc[a][0][k], acc[a][1][k], acc[a][2][k], acc[a][3][k]};
                } else {
#pragma unroll
                    for (int b = 0; b < 3; ++b)
                        if (ic + b < P.cols) to[b] = acc[a][b][k];
                }
            }
        if (leader) {
            float* sums = reinterpret_cast<float*>(&S.A[0][0][0][0]);  // [BO][8 groups of rows]; every wave is past its last step
            if (has_g) {
#pragma unroll
                for (int c = 0; c < 4; ++c) sums[(4 * gc + c) * 8 + gr / 4] = bsum[c];
            }
            __syncthreads();
            for (int q = tid; q < BO && o0 + q < P.out; q += THREADS) {
                const float* s = sums + q * 8;
                P.gb[(size_t)split * P.out + o0 + q] = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
            }
        }
    }
};

template <int TYPE, int BO, int BI, int WO, int WI, int MASK, bool NARROW>
__global__ void __launch_bounds__(64 * WO * WI, 2)
act_weight_grad_kernel(ActGrad P) {
    typedef WeightGrad<TYPE, BO, BI, WO, WI, MASK, NARROW> Pass;
    __shared__ __align__(16) typename Pass::Lds lds;
    // workgroups go to the eight XCDs in turn: the tiles of one split, which read the same rows, stay on one of them
    const int tiles = ((P.cols + BI - 1) / BI) * ((P.out + BO - 1) / BO);
    const int turn = blockIdx.x >> 3, split = (turn / tiles) * 8 + (blockIdx.x & 7);
    if (split >= P.splits) return;
    Pass pass{P, lds};
    pass.run(split, turn % tiles);
}

// Sums of the splits in double: the weight's entries, then the bias's.  A workgroup has 64 entries, its WAVES waves every
// WAVES-th split each, and their sums are added in order.
template <int WAVES>
__global__ void __launch_bounds__(64 * WAVES)
act_join_kernel(const float* __restrict__ part_w, const float* __restrict__ part_b, int64_t nw, int nb, int splits,
                float* __restrict__ gw, float* __restrict__ gb) {
    __shared__ double sums[WAVES][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t at = (int64_t)blockIdx.x * 64 + lane;
    const bool bias = at >= nw, live = at < nw + nb;
    const float* p = bias ? part_b + (at - nw) : part_w + at;
    const int64_t step = bias ? nb : nw;
    double s = 0.0;
    if (live)
#pragma unroll 8
        for (int k = wave; k < splits; k += WAVES) s += (double)p[k * step];
    sums[wave][lane] = s;
    __syncthreads();
    if (wave || !live) return;
    double all = 0.0;
#pragma unroll
    for (int k = 0; k < WAVES; ++k) all += sums[k][lane];
    if (bias) gb[at - nw] = (float)all;
    else gw[at] = (float)all;
}

// -------------------------------------------------------------------------------------------------------- column sums
//
//   sums[c] = sum_m x[m][c], the bias gradient of a layer whose activations were not kept in 8 bits.  (A library's sum that splits a
//   column over workgroups clears its counters with a memory-set call, and such a node of a captured graph does not do its work in
//   every replay; nothing here needs clearing.)
// A thread has four neighbouring columns of every (256 / groups)-th row of its split, sums in float32, a workgroup's threads are added
// in order in double, the splits by act_join_kernel.  Bound by memory where rows are many: 131072 x 512 float32 values in 50 us, 5.4 TB/s
// (the library's sum 89); 2048 x 512 in 5.6 us, two launches (11).

template <int TYPE>
__global__ void __launch_bounds__(256)
column_sums_kernel(const void* __restrict__ x, int64_t rows, int cols, int groups, int splits, float* __restrict__ part) {
    __shared__ float sums[256][4];
    __shared__ double fours[256];
    const int tid = threadIdx.x, each = 256 / groups, mine = tid / groups;  // groups of columns: a power of two up to 64
    const int c0 = (blockIdx.x * groups + (tid & (groups - 1))) * 4;
    float acc[4] = {0, 0, 0, 0};
    if (c0 + 4 <= cols) {
#pragma unroll 4
        for (int64_t m = (int64_t)blockIdx.y * each + mine; m < rows; m += (int64_t)splits * each) {
            float v[4];
            const int64_t at = m * cols + c0;
            if constexpr (TYPE == MARL_F32) {
                const f32x4 u = *reinterpret_cast<const f32x4_a4*>(static_cast<const float*>(x) + at);
                v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
            } else {
                typedef u32x2 u32x2_a2 __attribute__((aligned(2)));
                const u32x2 u = *reinterpret_cast<const u32x2_a2*>(static_cast<const uint16_t*>(x) + at);
                use_four<TYPE, false>(u32x4{u.x, u.y, 0, 0}, 0, v);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[k] += v[k];
        }
    } else if (c0 < cols) {
#pragma unroll 4
        for (int64_t m = (int64_t)blockIdx.y * each + mine; m < rows; m += (int64_t)splits * each)
#pragma unroll
            for (int k = 0; k < 3; ++k)
                if (c0 + k < cols) acc[k] += load_one<TYPE>(x, m * cols + c0 + k);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) sums[tid][k] = acc[k];
    __syncthreads();
    const int wide = 4 * groups, q = tid & (wide - 1), c = blockIdx.x * wide + q;  // a column of the tile, four rows of it to a thread
    double s = 0.0;
#pragma unroll
    for (int k = 0; k < 4; ++k) s += (double)sums[(tid / wide * 4 + k) * groups + q / 4][q & 3];
    fours[tid] = s;
    __syncthreads();
    if (tid >= wide || c >= cols) return;
    s = 0.0;
#pragma unroll 8
    for (int r = 0; r < 256; r += wide) s += fours[r + q];
    part[(int64_t)blockIdx.y * cols + c] = (float)s;
}

// ------------------------------------------------------------------------------------------------------------ host

// Tiles of up to 256 columns; a thread has at least eight rows, or up to 32 where that saves the second launch, and there are at most
// 1024 workgroups (131072 x 512: 512 splits).
struct SumsCut { int groups, tiles, splits; };
static SumsCut sums_cut(int64_t rows, int cols) {
    SumsCut c;
    c.groups = 1;
    while (c.groups < 64 && c.groups * 4 < cols) c.groups *= 2;
    c.tiles = (cols + c.groups * 4 - 1) / (c.groups * 4);
    const int64_t least = 8 * (256 / c.groups), most = rows <= 4 * least ? 1 : (rows + least - 1) / least, s = c.tiles >= 1024 ? 1 : 1024 / c.tiles;
    c.splits = (int)(s < most ? s : most);
    return c;
}

// How a weight gradient is cut: the tile, and into how many splits of the rows.  Measured in us (float32, with a mask):
//   out <= 16: tiles of 16 x 256 on two workgroups a compute unit; a split has at least 4 steps, where there are few rows 2
//     (65000 x 8 x 256: 15.6, with 8 steps 17.9, 2 steps 19.7; 2048 x 8 x 256: 7.6, with 8 steps 17.6)
//   otherwise tiles of 128 x 256 on one workgroup a compute unit where there is work for them with 4 steps a split (8192 x 512 x
//     202: 24.5, with small tiles 28.5), else 64 x 64 on two with 4 steps (2048 x 512 x 202: 14.5; 2 steps 18.5, 8 steps 15.8),
//     and for inputs that one of those covers: the gradient is then read once, and x, the smaller operand, once for every 64 outputs
//     (131072 x 512 x 40: 123 and 132, without a mask x 64: 81 and 107; with two of them it is slower, x 96: 186 and 134)
// Two sizes are slow, though right: 17 to 64 outputs of more than 64 inputs multiply outputs that are not there (131072 x 20 x 512: 52
// us, 15 of bytes), and weights of so many tiles that there are fewer than eight splits leave XCDs without work, since a split's tiles
// stay on one (131072 x 2048 x 2048, two splits: 10.6 ms; 1024 x 1024, eight: 0.8).
struct ActCut { int bo, bi, splits; int64_t grid; };
static ActCut act_cut(int64_t rows, int out, int cols) {
    ActCut c;
    const int64_t steps = (rows + WG_STEP - 1) / WG_STEP;
    const auto tiles = [&](int bo, int bi) { return (int64_t)((out + bo - 1) / bo) * ((cols + bi - 1) / bi); };
    if (out <= 16 || cols < 4) { c.bo = 16; c.bi = 256; }
    else if (cols > 64 && tiles(128, 256) * (steps / 4) >= 256) { c.bo = 128; c.bi = 256; }
    else { c.bo = 64; c.bi = 64; }
    const int64_t t = tiles(c.bo, c.bi);
    int64_t s = (c.bo == 128 ? 256 : 512) / t;
    s = s < 1 ? 1 : s;
    const int64_t least = c.bo == 16 ? (steps > 512 ? 4 : 2) : 4, most = (steps + least - 1) / least;
    s = s > most ? most : s;
    const int64_t each = (steps + s - 1) / s;
    c.splits = (int)((steps + each - 1) / each);
    c.grid = (int64_t)(c.splits + 7) / 8 * 8 * t;
    return c;
}

template <int TYPE, int MASK>
static void launch_weight_grad_mask(const ActGrad& P, const ActCut& c, hipStream_t stream) {
    const dim3 grid((uint32_t)c.grid);
    if (c.bo == 16 && (P.out < 4 || P.cols < 4))
        hipLaunchKernelGGL((act_weight_grad_kernel<TYPE, 16, 256, 1, 4, MASK, true>), grid, dim3(256), 0, stream, P);
    else if (c.bo == 16) hipLaunchKernelGGL((act_weight_grad_kernel<TYPE, 16, 256, 1, 4, MASK, false>), grid, dim3(256), 0, stream, P);
    else if (c.bo == 64) hipLaunchKernelGGL((act_weight_grad_kernel<TYPE, 64, 64, 4, 1, MASK, false>), grid, dim3(256), 0, stream, P);
    else hipLaunchKernelGGL((act_weight_grad_kernel<TYPE, 128, 256, 2, 4, MASK, false>), grid, dim3(512), 0, stream, P);
}
template <int TYPE>
static void launch_weight_grad_type(const ActGrad& P, const ActCut& c, hipStream_t stream) {
    if (!P.mask) launch_weight_grad_mask<TYPE, UNCUT>(P, c, stream);
    else if (P.masked) launch_weight_grad_mask<TYPE, CUT_KEPT>(P, c, stream);
    else launch_weight_grad_mask<TYPE, CUT>(P, c, stream);
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
    if (too_many_blocks(num_rows, num_cols)) return set_error(MARL_ERR_INVALID, "more than 2^30 - 64 blocks of 32 values in one call");
    const int blocks = (int)lb_blocks(num_cols);
    const auto pick = [&](auto positive, auto nt) {
        constexpr bool pos = decltype(positive)::value, hint = decltype(nt)::value;
        return x_type == MARL_F32 ? act_compress_kernel<MARL_F32, pos, hint> : x_type == MARL_BF16 ? act_compress_kernel<MARL_BF16, pos, hint>
                                                                                                   : act_compress_kernel<MARL_F16, pos, hint>;
    };
    const auto yes = std::true_type{};
    const auto no = std::false_type{};
    const bool nt = (uint64_t)num_rows * num_cols * lb_type_bytes(x_type) > LB_NT_BYTES;
    auto kernel = nonnegative ? (nt ? pick(yes, yes) : pick(yes, no)) : (nt ? pick(no, yes) : pick(no, no));
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
    if (too_many_blocks(num_rows, num_cols)) return set_error(MARL_ERR_INVALID, "more than 2^30 - 64 blocks of 32 values in one call");
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

// Both entry points: `keep` says whether the cut gradient is a result.
static int weight_grad(bool keep, const void* d_grad, int grad_type, int64_t num_rows, int num_out, const uint8_t* d_codes,
                       const uint8_t* d_scales, int num_cols, int nonnegative, const uint8_t* d_mask_codes, void* d_masked_grad,
                       float* d_grad_weight, float* d_grad_bias, void* d_workspace, void* stream) {
    if (num_rows <= 0 || num_out <= 0 || num_cols <= 0)
        return set_error(MARL_ERR_INVALID, "num_rows, num_out and num_cols must be positive");
    if (grad_type != MARL_F32 && grad_type != MARL_BF16 && grad_type != MARL_F16)
        return set_error(MARL_ERR_INVALID, "grad_type must be MARL_F32, MARL_BF16 or MARL_F16");
    if (!d_grad || !d_codes || !d_scales || !d_grad_weight || !d_grad_bias)
        return set_error(MARL_ERR_INVALID, keep ? "NULL argument to marl_act_weight_grad" : "NULL argument to marl_act_param_grad");
    if (keep && (d_mask_codes == nullptr) != (d_masked_grad == nullptr))
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
    P.splits = c.splits;
    P.gw = c.splits == 1 ? d_grad_weight : static_cast<float*>(d_workspace);
    P.gb = c.splits == 1 ? d_grad_bias : static_cast<float*>(d_workspace) + c.splits * nw;
    if (grad_type == MARL_F32) launch_weight_grad_type<MARL_F32>(P, c, s);
    else if (grad_type == MARL_BF16) launch_weight_grad_type<MARL_BF16>(P, c, s);
    else launch_weight_grad_type<MARL_F16>(P, c, s);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || c.splits == 1) return act_hip(e, "weight gradient launch");
    const int64_t groups = (nw + num_out + 63) / 64;
    // where the entries leave half of the compute units empty, four times the waves to each (65000 x 8 x 256: 17.9 against 20.0)
    const bool few = groups < 128;
    hipLaunchKernelGGL(few ? act_join_kernel<16> : act_join_kernel<4>, dim3((uint32_t)groups), dim3(few ? 1024 : 256), 0, s, P.gw, P.gb, nw,
                       num_out, c.splits, d_grad_weight, d_grad_bias);
    return act_hip(hipGetLastError(), "weight gradient join launch");
}

extern "C" int marl_act_weight_grad(const void* d_grad, int grad_type, int64_t num_rows, int num_out, const uint8_t* d_codes,
                                    const uint8_t* d_scales, int num_cols, int nonnegative, const uint8_t* d_mask_codes,
                                    void* d_masked_grad, float* d_grad_weight, float* d_grad_bias, void* d_workspace, void* stream) {
    return weight_grad(true, d_grad, grad_type, num_rows, num_out, d_codes, d_scales, num_cols, nonnegative, d_mask_codes, d_masked_grad,
                       d_grad_weight, d_grad_bias, d_workspace, stream);
}

extern "C" int marl_act_param_grad(const void* d_grad, int grad_type, int64_t num_rows, int num_out, const uint8_t* d_codes,
                                   const uint8_t* d_scales, int num_cols, int nonnegative, const uint8_t* d_mask_codes,
                                   float* d_grad_weight, float* d_grad_bias, void* d_workspace, void* stream) {
    return weight_grad(false, d_grad, grad_type, num_rows, num_out, d_codes, d_scales, num_cols, nonnegative, d_mask_codes, nullptr,
                       d_grad_weight, d_grad_bias, d_workspace, stream);
}

extern "C" size_t marl_column_sums_workspace_bytes(int64_t num_rows, int num_cols) {
    if (num_rows <= 0 || num_cols <= 0) return 0;
    const SumsCut c = sums_cut(num_rows, num_cols);
    return c.splits == 1 ? 0 : (size_t)c.splits * num_cols * sizeof(float);
}

extern "C" int marl_column_sums(const void* d_x, int x_type, int64_t num_rows, int num_cols, float* d_sums, void* d_workspace, void* stream) {
    if (num_rows <= 0 || num_cols <= 0) return set_error(MARL_ERR_INVALID, "num_rows and num_cols must be positive");
    if (x_type != MARL_F32 && x_type != MARL_BF16 && x_type != MARL_F16)
        return set_error(MARL_ERR_INVALID, "x_type must be MARL_F32, MARL_BF16 or MARL_F16");
    if (!d_x || !d_sums) return set_error(MARL_ERR_INVALID, "NULL argument to marl_column_sums");
    if (((uintptr_t)d_x & (lb_type_bytes(x_type) - 1)) != 0 || ((uintptr_t)d_sums & 3u) != 0 || ((uintptr_t)d_workspace & 15u) != 0)
        return set_error(MARL_ERR_INVALID, "d_workspace must be 16-byte aligned, the others aligned to their elements");
    if (num_rows >= ((int64_t)1 << 40) || num_cols > (1 << 20)) return set_error(MARL_ERR_INVALID, "at most 2^40 rows and 2^20 columns");
    const SumsCut c = sums_cut(num_rows, num_cols);
    if (c.splits > 1 && !d_workspace)
        return set_error(MARL_ERR_INVALID, "this size needs d_workspace (marl_column_sums_workspace_bytes bytes)");
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    float* part = c.splits == 1 ? d_sums : static_cast<float*>(d_workspace);
    auto kernel = x_type == MARL_F32 ? column_sums_kernel<MARL_F32> : x_type == MARL_BF16 ? column_sums_kernel<MARL_BF16> : column_sums_kernel<MARL_F16>;
    hipLaunchKernelGGL(kernel, dim3(c.tiles, c.splits), dim3(256), 0, s, d_x, num_rows, num_cols, c.groups, c.splits, part);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || c.splits == 1) return act_hip(e, "column sums launch");
    hipLaunchKernelGGL(act_join_kernel<16>, dim3((uint32_t)((num_cols + 63) / 64)), dim3(1024), 0, s, part, part, (int64_t)0, num_cols, c.splits, d_sums, d_sums);
    return act_hip(hipGetLastError(), "column sums join launch");
}
