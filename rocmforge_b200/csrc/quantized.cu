// Weights in 4 bits and rows in 8 bits: the products of few tokens that read them, and what makes such weights and rows.
//
// Weights: w[n, k] = s[n, k / G] q[n, k], q in -8..7 and s bfloat16, groups of G = 32, 64 or 128 columns.  Rows: x[t, k] =
// a[t, k / G] p[t, k], p in -127..127 and a = max|x| / 127 of the group in float32.  maeddesg/ROCmForge's products of Q4_0 and Q4_1
// blocks with Q8_0 rows (hip_kernels/quant/, src/gpu/quant_wrapper.rs) use the same pair, blocks of 32 and halves as scales; the layout,
// the group sizes and the kernels here are this library's own.
//
// How weights are stored: quantized.cuh.
#include "quantized.cuh"
#include <type_traits>

template <typename T> struct Quad;                       // four neighbouring numbers
template <> struct Quad<float> {
    static __device__ __forceinline__ void load(const float* p, float* v) {
        const float4 x = *reinterpret_cast<const float4*>(p);
        v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
    }
};
template <> struct Quad<__nv_bfloat16> {
    static __device__ __forceinline__ void load(const __nv_bfloat16* p, float* v) {
        const uint2 x = *reinterpret_cast<const uint2*>(p);
        v[0] = __uint_as_float(x.x << 16); v[1] = __uint_as_float(x.x & 0xffff0000u);
        v[2] = __uint_as_float(x.y << 16); v[3] = __uint_as_float(x.y & 0xffff0000u);
    }
};
// Columns c .. c + 3 of a row of n numbers, zeros from n on.  VEC: the row starts on an access of four and n is a multiple of four.
template <typename T, bool VEC>
__device__ __forceinline__ void load_quad(const T* row, int c, int n, float* v) {
    if constexpr (VEC) {
        if (c < n) Quad<T>::load(row + c, v);
        else v[0] = v[1] = v[2] = v[3] = 0.f;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = c + i < n ? Cvt<T>::to_f32(row[c + i]) : 0.f;
    }
}

__device__ __forceinline__ float max_nan(float a, float b) {           // NaN if either is
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
    return m;
}

// The 8-bit form of a group: G / 4 neighbouring lanes hold four numbers each; returns the lane's four bytes, and the group's scale in
// `scale`.  A group of zeros has the scale 0, one below 2^-120 too (127 / m must stay finite); a NaN or an infinity in a group makes its
// scale NaN, so that every product that reads it is NaN, as one of the numbers themselves would be NaN or infinite.
template <int G>
__device__ __forceinline__ uint32_t to_8_bits(const float* v, float& scale) {
    float m = max_nan(max_nan(fabsf(v[0]), fabsf(v[1])), max_nan(fabsf(v[2]), fabsf(v[3])));
#pragma unroll
    for (int o = G / 8; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    const bool finite = m < INFINITY, some = m >= 0x1p-120f;
    scale = !finite ? __uint_as_float(0x7fffffffu) : some ? m / 127.f : 0.f;
    if (!finite || !some) return 0u;
    const float inv = 127.f / m;                          // |v| inv <= 127 (1 + 2^-23): rounds to 127 at most
    uint32_t out = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) out |= (uint32_t)(__float2int_rn(v[i] * inv) & 255) << (8 * i);
    return out;
}

// Where a thread of a block of 256 is that has EACH columns at a time: narrow rows share a block (`across` of them), wide ones take several.
template <int EACH>
struct Place {
    int across, sub, c;                                  // (a thread without a row of its own: columns behind the last)
    __device__ __forceinline__ Place(int Kp) {
        const int units = Kp / EACH;
        across = units < 256 ? 256 / units : 1;
        sub = units < 256 ? threadIdx.x / units : 0;
        c = units < 256 ? (sub < across ? EACH * (threadIdx.x - sub * units) : Kp) : EACH * (blockIdx.x * 256 + threadIdx.x);
    }
};

// ---------------------------------------------------------------- rows to 8 bits
// A lane has four columns.  (64 x 3,584 1.6 us: a launch; 2,048 x 3,584 10.8, floor 3.4: a group's two divisions and shuffles in every lane.)
template <typename T, int G, bool VEC>
__global__ void __launch_bounds__(256) quantize_q8_kernel(const T* x, long long ldx, int8_t* __restrict__ q, float* __restrict__ scales,
                                                          int T_, int K, int Kp) {
    pdl_trigger();
    pdl_wait(x);
    const Place<4> at(Kp);
    for (int t0 = blockIdx.y * at.across; t0 < T_; t0 += gridDim.y * at.across) {
        const int t = t0 + at.sub, c = t < T_ ? at.c : Kp;               // (all lanes of a group do the same)
        float v[4], s;
        load_quad<T, VEC>(x + (size_t)t * ldx, c, K, v);
        const uint32_t p = to_8_bits<G>(v, s);
        if (c < Kp) {
            *reinterpret_cast<uint32_t*>(q + (size_t)t * Kp + c) = p;
            if (c % G == 0) scales[(size_t)t * (Kp / G) + c / G] = s;
        }
    }
}

// ... and the numbers that 8-bit rows stand for, eight (rows of whole eights, on 16-byte boundaries: 2,048 x 3,584 5.9 us, by fours 9.2) or four
// columns a thread.
template <typename T, int EACH>
__global__ void __launch_bounds__(256) dequantize_q8_kernel(const int8_t* q, const float* scales, T* __restrict__ y, int T_, int K, int Kp, int G) {
    pdl_trigger();
    pdl_wait(q, scales);
    const Place<EACH> at(Kp);
    const int c = at.c;
    if (c >= K) return;
    for (int t = blockIdx.y * at.across + at.sub; t < T_; t += gridDim.y * at.across) {
        const float s = scales[(size_t)t * (Kp / G) + c / G];
        T* to = y + (size_t)t * K + c;
        if constexpr (EACH == 8) {
            const uint2 p = *reinterpret_cast<const uint2*>(q + (size_t)t * Kp + c);
            __align__(16) T v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = Cvt<T>::from_f32((float)(int8_t)((i < 4 ? p.x : p.y) >> (8 * (i & 3))) * s);
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(to)[i] = reinterpret_cast<const uint4*>(v)[i];
        } else {
            const char4 p = *reinterpret_cast<const char4*>(q + (size_t)t * Kp + c);
            const float v[4] = {p.x * s, p.y * s, p.z * s, p.w * s};
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (c + i < K) to[i] = Cvt<T>::from_f32(v[i]);
        }
    }
}

// ---------------------------------------------------------------- gated unit to 8 bits
// y[t, j] = act(gu[t, 2j]) gu[t, 2j + 1] (the fused weight's rows are interleaved), in 32 bits and from there to 8.  gelu by tanh, 0.5 g (1 + tanh(u)),
// is g / (1 + exp(-2 u)): 1 + tanh(u) loses its bits where a gate is far below zero (30 % at -5, everything at -5.6), and such a group's scale
// comes from those values.  128 x 18,944 gelu 6.5 us (from
// 32-bit sums 6.7; rounded to 16 bits instead 4.9): exponentials, divisions and four bytes a lane; 1 x 4,864 1.7: a launch.
template <typename T, int ACT, int G, bool VEC>
__global__ void __launch_bounds__(256) swiglu_q8_kernel(const T* gu, int8_t* __restrict__ q, float* __restrict__ scales, int T_, int I, int Ip) {
    pdl_trigger();
    pdl_wait(gu);
    const Place<4> at(Ip);
    for (int t0 = blockIdx.y * at.across; t0 < T_; t0 += gridDim.y * at.across) {
        const int t = t0 + at.sub, c = t < T_ ? at.c : Ip;
        const T* row = gu + (size_t)t * 2 * I;
        float a[4], b[4], v[4], s;
        load_quad<T, VEC>(row, 2 * c, 2 * I, a);
        load_quad<T, VEC>(row, 2 * c + 4, 2 * I, b);
        const float g[4] = {a[0], a[2], b[0], b[2]}, u[4] = {a[1], a[3], b[1], b[3]};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float act;
            if constexpr (ACT == 0) act = g[i] / (1.f + expf(-g[i]));
            else if constexpr (ACT == 1) act = fmaxf(g[i], 0.f);
            else act = g[i] / (1.f + expf(-1.5957691216057308f * (g[i] + 0.044715f * g[i] * g[i] * g[i])));
            v[i] = act * u[i];
        }
        const uint32_t p = to_8_bits<G>(v, s);
        if (c < Ip) {
            *reinterpret_cast<uint32_t*>(q + (size_t)t * Ip + c) = p;
            if (c % G == 0) scales[(size_t)t * (Ip / G) + c / G] = s;
        }
    }
}

// ---------------------------------------------------------------- add + RMSNorm to 8 bits
// v = h[row] + sum_s pending[s][row];  y = v rsqrt(mean(v^2) + eps) w, to 8 bits from 32.  The kinds of pending and of rows are those
// of add_rmsnorm (elementwise.cu).  A block has a row, a lane four columns at a time, in registers: one pass over the stream and what is added to
// it.  2,048 x 3,584 after a 16-bit update 17.4 us, 4.7 TB/s (the norm with a 16-bit result 21.1); 64 x 5,120 after five sums 4.7 and 1 x 896 after
// four 2.1: a chain of trips to L2 and of the block's sum.
template <typename T, int G, int NV, bool VEC>
__global__ void __launch_bounds__(1024) add_rmsnorm_q8_kernel(float* __restrict__ h, const void* pending, int kind, int n_pending,
                                                              size_t pstride, const void* w, int w_is_f32, float eps,
                                                              int8_t* __restrict__ q, float* __restrict__ scales, const int* rows, int n_h, int H, int Hp) {
    pdl_trigger();
    __shared__ float red[34];
    const int r = blockIdx.x;
    pdl_wait(pending, rows);                             // (rows may be what the kernel before has just chosen)
    const int t = rows ? min(max(rows[r], 0), n_h - 1) : r;             // (a row that is not there is never read)
    float* hrow = h + (size_t)t * H;
    float v[NV][4];
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = 4 * (threadIdx.x + i * blockDim.x);
        load_quad<float, VEC>(hrow, c, H, v[i]);
        if (kind == 1) {
#pragma unroll 4                                        // (loads before sums)
            for (int s = 0; s < n_pending; ++s) {
                float p[4];
                load_quad<float, VEC>(reinterpret_cast<const float*>(pending) + (size_t)s * pstride + (size_t)t * H, c, H, p);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[i][j] += p[j];
            }
        } else if (kind == 2) {
            float p[4];
            load_quad<T, VEC>(reinterpret_cast<const T*>(pending) + (size_t)t * H, c, H, p);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[i][j] += p[j];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) ss += v[i][j] * v[i][j];
    }
    const float inv = rsqrtf(block_sum(ss, red) / (float)H + eps);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = 4 * (threadIdx.x + i * blockDim.x);
        if (!rows && kind != 0) {
            if constexpr (VEC) {
                if (c < H) *reinterpret_cast<float4*>(hrow + c) = make_float4(v[i][0], v[i][1], v[i][2], v[i][3]);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (c + j < H) hrow[c + j] = v[i][j];
            }
        }
        float y[4], s;
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = c + j < H ? v[i][j] * inv * load_vec(w, w_is_f32, c + j) : 0.f;
        const uint32_t p = to_8_bits<G>(y, s);
        if (c < Hp) {
            *reinterpret_cast<uint32_t*>(q + (size_t)r * Hp + c) = p;
            if (c % G == 0) scales[(size_t)r * (Hp / G) + c / G] = s;
        }
    }
}

// ---------------------------------------------------------------- weights to 4 bits, and back
// The scale of a group: its largest magnitude becomes 7.5 steps (a grid of -8..7 then misses it by 3/4 of a step at most), rounded to five
// significant bits.  s q has at most eight then, so every weight is a bfloat16 number: the products of 8-bit rows and the 16-bit products
// of a prompt multiply the same weights, and nothing is rounded between them.  Steps of 1/16 octave between scales cost 3 % of the
// quantisation step at most.  A NaN or an infinity makes the group's scale NaN.
__device__ __forceinline__ float w4_scale(float m) {
    if (!(m < INFINITY)) return __uint_as_float(0x7fc00000u);
    if (m < 0x1p-100f) return 0.f;
    uint32_t u = __float_as_uint(m / 7.5f);
    u += 0x3ffffu + (u >> 19 & 1u);                      // to the nearest of five significant bits, ties to even
    return __uint_as_float(u & 0xfff80000u);
}
// A warp makes the tiles of a group's columns: lane 4 g + t holds the eight columns of its two rows and two halves, 32 numbers a tile, read one by
// one (rows start anywhere).  37,888 x 3,584 150 us from float32, 4.1 TB/s, 179 from bfloat16: loads; it runs once, when a model is made.
template <typename T, int G>
__global__ void __launch_bounds__(256) quantize_w4_kernel(const T* weight, long long ldw, uint4* __restrict__ packed, __nv_bfloat16* __restrict__ scales,
                                                          int N, int K, int Kp) {
    constexpr int TILES = G == 128 ? 2 : 1;              // tiles of 64 columns that a group spans
    constexpr int GROUPS = G == 32 ? 2 : 1;              // groups in that many columns
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int units = Kp / (64 * TILES);
    const long long unit = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (unit >= (long long)((N + 15) / 16) * units) return;
    const int tile = (int)(unit / units), col0 = (int)(unit % units) * 64 * TILES;
    float m[2][GROUPS] = {}, v[TILES][2][2][8];
#pragma unroll
    for (int b = 0; b < TILES; ++b)
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int n = 16 * tile + g + 8 * r, k = col0 + 64 * b + 32 * c + 8 * t + j;
                    v[b][r][c][j] = n < N && k < K ? Cvt<T>::to_f32(weight[(size_t)n * ldw + k]) : 0.f;
                    m[r][GROUPS == 2 ? c : 0] = max_nan(m[r][GROUPS == 2 ? c : 0], fabsf(v[b][r][c][j]));
                }
    float s[2][GROUPS], inv[2][GROUPS];
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int c = 0; c < GROUPS; ++c) {
            m[r][c] = max_nan(m[r][c], __shfl_xor_sync(0xffffffffu, m[r][c], 1));
            m[r][c] = max_nan(m[r][c], __shfl_xor_sync(0xffffffffu, m[r][c], 2));
            s[r][c] = w4_scale(m[r][c]);
            inv[r][c] = s[r][c] > 0.f ? 1.f / s[r][c] : 0.f;             // (a NaN scale leaves zeros behind it)
            if (t == 0) scales[((size_t)tile * (Kp / G) + col0 / G + c) * 16 + 2 * g + r] = __float2bfloat16_rn(s[r][c]);
        }
#pragma unroll
    for (int b = 0; b < TILES; ++b) {
        uint32_t word[4];
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                word[2 * r + c] = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float f = inv[r][GROUPS == 2 ? c : 0];
                    const int i = f > 0.f ? max(-8, min(7, __float2int_rn(v[b][r][c][j] * f))) : 0;
                    word[2 * r + c] |= (uint32_t)(i & 15) << (8 * (j & 3) + 4 * (j >> 2));
                }
            }
        packed[((size_t)tile * (Kp / 64) + col0 / 64 + b) * 32 + lane] = make_uint4(word[0], word[1], word[2], word[3]);
    }
}

// The weights as numbers, columns lo .. hi - 1 (lo a multiple of 64): a warp writes a tile, a lane four runs of eight columns.  37,888 x 3,584 to
// bfloat16 56 us, 6.1 TB/s, to float32 134 us, 4.6 TB/s: what it writes.
template <typename T, int G>
__global__ void __launch_bounds__(256) dequantize_w4_kernel(const uint4* packed, const __nv_bfloat16* scales, T* __restrict__ out, int N, int Kp, int lo, int hi) {
    pdl_wait(packed, scales);
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, blocks = (hi - lo + 63) / 64;
    const long long unit = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (unit >= (long long)((N + 15) / 16) * blocks) return;
    const int tile = (int)(unit / blocks), k0 = lo + 64 * (int)(unit % blocks), ld = hi - lo;
    const uint4 p = packed[((size_t)tile * (Kp / 64) + k0 / 64) * 32 + lane];
    const uint32_t word[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int n = 16 * tile + g + 8 * r, k = k0 + 32 * c + 8 * t;
            if (n >= N || k >= hi) continue;
            const float s = __bfloat162float(scales[((size_t)tile * (Kp / G) + k / G) * 16 + 2 * g + r]);
            alignas(16) T v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int i = (int)(word[2 * r + c] >> (8 * (j & 3) + 4 * (j >> 2)) & 15u);
                v[j] = Cvt<T>::from_f32((float)((i ^ 8) - 8) * s);
            }
            T* to = out + (size_t)n * ld + (k - lo);
            if (ld % 8 == 0) {
#pragma unroll
                for (int j = 0; j < 8 * (int)sizeof(T) / 16; ++j) reinterpret_cast<uint4*>(to)[j] = reinterpret_cast<const uint4*>(v)[j];
            } else {
                for (int j = 0; j < 8 && k + j < hi; ++j) to[j] = v[j];
            }
        }
}

// Products stream their weights before they wait for the kernel before them, which holds for weights that were there before the step.
// Where a kernel has just made them, this one stands between: it is launched without the early start, so what was written before it is
// complete and visible when it begins, and the product's early part begins no sooner.
__global__ void weights_made_kernel() {}

// ---------------------------------------------------------------- products of few tokens
// d = A B + c, A 16 rows by 32 (16) columns of weights, B as many columns by eight tokens.
__device__ __forceinline__ void mma_s8(int (&d)[4], const int* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(c[0]), "r"(c[1]), "r"(c[2]), "r"(c[3]));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
// d = (rows g, g + 8; 32 columns) times the token's numbers + c: a word of four bytes a row, eight numbers.
__device__ __forceinline__ void quarter(int (&d)[4], const int* c, uint32_t lo_row, uint32_t hi_row, const uint2& x) {
    const uint32_t m = 0xf0f0f0f0u;                      // a half of a byte at its upper end is 16 q as a signed byte
    mma_s8(d, c, lo_row << 4 & m, hi_row << 4 & m, lo_row & m, hi_row & m, x.x, x.y);
}
// Two bytes q + 8 below 0x43 each are 128 + q + 8, less 136; exact.
__device__ __forceinline__ uint32_t two_weights(uint32_t bytes, uint32_t which) {
    uint32_t v = __byte_perm(bytes, 0x43434343u, which);
    const __nv_bfloat162 less = __float2bfloat162_rn(-136.f);
    __nv_bfloat162 r = __hadd2(*reinterpret_cast<__nv_bfloat162*>(&v), less);
    return *reinterpret_cast<uint32_t*>(&r);
}
__device__ __forceinline__ void quarter(float (&d)[4], const float* c, uint32_t lo_row, uint32_t hi_row, const uint4& x) {
    const uint32_t m = 0x0f0f0f0fu, eight = 0x08080808u;
    const uint32_t l0 = (lo_row & m) ^ eight, h0 = (hi_row & m) ^ eight, l1 = (lo_row >> 4 & m) ^ eight, h1 = (hi_row >> 4 & m) ^ eight;
    mma_bf16(d, c, two_weights(l0, 0x4140), two_weights(h0, 0x4140), two_weights(l0, 0x4342), two_weights(h0, 0x4342), x.x, x.y);
    mma_bf16(d, d, two_weights(l1, 0x4140), two_weights(h1, 0x4140), two_weights(l1, 0x4342), two_weights(h1, 0x4342), x.z, x.w);
}
__device__ __forceinline__ unsigned long long two(float a, float b) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ unsigned long long add_two(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ unsigned long long mul_two(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ unsigned long long fma_two(unsigned long long a, unsigned long long b, unsigned long long c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// 8 NB tokens (blockIdx.y) by tiles of 16 RT rows, one block of 16 warps an SM for as long as there are tiles.  With RT = 2 a token's numbers,
// once in registers, meet 32 rows: from two eights of tokens on the reads of shared memory would otherwise take longer than the products.  The numbers of the block's
// tokens lie in shared memory from the start (a cluster's CTAs have a share of the columns each, so that they fit), and their scales.  A
// warp goes through its tiles in units of 128 columns (1 KB of weights), which asynchronous copies bring into a ring of its own, DEPTH
// units ahead and without regard to where a tile ends; a lane reads back what it has copied itself (but for the scales).  No
// warp waits for another but once a round, when `ways` warps (and the cluster's CTAs) add up what they have of a tile, and not even then
// where a tile is one warp's.
// A group's (at most 128 columns') exact sum is formed by the tensor cores in whole numbers and added up in 32 bits; the whole number starts
// at 1.5 2^23 as a float's bits, so that its bits are that float plus the sum (below 2^22: 128 columns of 16 * 8 * 127), and no conversion is
// needed.  16-bit rows: the halves of bytes become bfloat16 numbers and a group's sum is a float.
// What bounds it, and what it took (device time in a chain of launches over weights larger than L2): 1 to 8 8-bit rows x 37,888 x 3,584 12.9 to
// 13.0 us, 5.4 TB/s: the weights' stream; 1 x 4,608 x 3,584 4.3 us, 1 x 896 x 896 2.4: a launch, one trip to memory and the warps' sums.  16 rows
// 14.0 us, 32 22.1, 64 39.2 (in groups of 32 columns 63; four eights of tokens by two tiles a warp, which the cost rule misses here, 34.5),
// 64 x 3,584 x 18,944 in groups of 64 32.8: instructions; at 64 x 37,888 x 3,584 the
// schedulers issue in 61 % of cycles and the tensor cores are busy in 39 %.  16-bit rows: 1 x 37,888 x
// 3,584 19 us, 16 x 27,648 x 5,120 27.0: widening the weights, whatever the tokens.
#define W4_WARPS 16
#define W4_SLOT (1024 + 128)                             // a unit's weights, and its scales [group][16 rows]
#define W4_SUMS(rt) (16 * (rt) * W4_WARPS + 4)           // pitch of the warps' sums [token][16 rt rows a warp]
// Shared memory of a block: tokens' numbers (rows a pitch apart by which eight tokens' reads meet every bank once), their scales
// [group][token], the warps' sums (two sets for a cluster that has several rounds, none where a tile is one warp's), the rings.
struct W4Shared {
    int columns, pitch, scales, sums, ring, bytes;
};
__host__ __device__ constexpr int w4_depth(int nb, int rt) { return nb == 1 ? 6 : nb == 2 ? 4 / rt + (rt - 1) : 3 - (rt - 1); }
__host__ __device__ inline int w4_rounds(int N, int rt, int ways, int clusters) {
    const int tiles = ((N + 15) / 16 + rt - 1) / rt, at_once = W4_WARPS / ways * clusters;
    return (tiles + at_once - 1) / at_once;
}
__host__ __device__ inline W4Shared w4_shared(int units, int rounds, int ways, int splits, int G, int size, int M, int nb, int rt) {
    W4Shared s;
    s.columns = (units + splits - 1) / splits * 128;
    s.pitch = s.columns * size + (size == 1 ? 32 : 64);
    s.scales = (M < 8 * nb ? M : 8 * nb) * s.pitch;
    s.sums = s.scales + (size == 1 ? s.columns / G * 8 * nb * 4 : 0);
    s.ring = s.sums + (splits > 1 && rounds > 1 ? 2 : splits > 1 || ways > 1 ? 1 : 0) * 8 * nb * W4_SUMS(rt) * 4;
    s.bytes = s.ring + W4_WARPS * w4_depth(nb, rt) * rt * W4_SLOT;
    return s;
}

template <int G, typename X, int NB, int RT>
__global__ void __launch_bounds__(32 * W4_WARPS, 1) w4_product_kernel(const uint4* __restrict__ w0, const uint32_t* __restrict__ w1, const X* x,
                                                                      const float* xs, long long ldx, int whole, int K, int blocks, int ways, int splits, W4Out o) {
    constexpr bool BYTES = std::is_same<X, int8_t>::value;
    constexpr int DEPTH = w4_depth(NB, RT), GROUPS = 128 / G, QUARTERS = G / 32, THREADS = 32 * W4_WARPS, SLOT = RT * W4_SLOT, SUMS = W4_SUMS(RT);
    extern __shared__ __align__(128) uint8_t smem[];
    pdl_trigger();
    const int units = (blocks + 1) / 2, all_groups = blocks * 64 / G;
    const uint32_t base = (uint32_t)__cvta_generic_to_shared(smem);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int rank = blockIdx.x % splits, cluster = blockIdx.x / splits, clusters = gridDim.x / splits;
    const int tiles16 = (o.N + 15) / 16, tiles = (tiles16 + RT - 1) / RT, at_once = W4_WARPS / ways, rounds = w4_rounds(o.N, RT, ways, clusters);
    const W4Shared sh = w4_shared(units, rounds, ways, splits, G, (int)sizeof(X), o.M, NB, RT);
    const int tok0 = blockIdx.y * 8 * NB, live = min(8 * NB, o.M - tok0);
    const int first = (int)((long long)units * rank / splits), count = (int)((long long)units * (rank + 1) / splits) - first;
    const int from = first + count * (warp % ways) / ways, to = first + count * (warp % ways + 1) / ways;
    auto tile_of = [&](int round) { return (round * clusters + cluster) * at_once + warp / ways; };
    // the unit that is asked for next, and the ring
    int ask_round = from < to && tile_of(0) < tiles ? 0 : rounds, ask_left = to - from;
    const uint32_t ring = base + sh.ring + warp * DEPTH * SLOT;
    uint32_t ask_to = ring + 16 * lane;
    const uint4* pw[RT];
    const uint32_t* ps[RT];
    auto start_tile = [&]() {
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            const int tile = min(RT * tile_of(ask_round) + r, tiles16 - 1);             // (rows that are not there: some others)
            pw[r] = w0 + ((size_t)tile * blocks + 2 * from) * 32 + lane;
            ps[r] = w1 + ((size_t)tile * all_groups + from * GROUPS + t) * 8 + g;
        }
    };
    start_tile();
    const bool half_last = (blocks & 1) && to == units;  // a row's last unit is its first half only: zeros, scales too, for the other
    const uint32_t scale_at = 1024 + 4 * (8 * t + g) - 16 * lane;
    auto ask = [&]() {
        if (ask_round < rounds) {
            const bool second = !(half_last && ask_left == 1);
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                copy16(ask_to + r * W4_SLOT, pw[r], true);
                copy16(ask_to + r * W4_SLOT + 512, second ? pw[r] + 32 : pw[r], second);
                const bool there = second || 2 * t < GROUPS;
                copy4_if(ask_to + r * W4_SLOT + scale_at, there ? ps[r] : w1, there, t < GROUPS);
                pw[r] += 64;
                ps[r] += 8 * GROUPS;
            }
            if (--ask_left == 0) {
                ask_left = to - from;
                if (tile_of(++ask_round) >= tiles) ask_round = rounds;
                else start_tile();
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        ask_to = ask_to == ring + 16 * lane + (DEPTH - 1) * SLOT ? ring + 16 * lane : ask_to + SLOT;
    };
    for (int i = 0; i < DEPTH; ++i) ask();
    pdl_wait(x, xs);
    if (whole) {
        constexpr int EACH = 16 / (int)sizeof(X);
        for (int tok = warp; tok < live; tok += W4_WARPS) {
            const X* row = x + (size_t)(tok0 + tok) * ldx;
            for (int i = lane; i < count * 128 / EACH; i += 32) {
                const int k = first * 128 + i * EACH;
                const bool there = k < (BYTES ? 64 * blocks : K);       // (16-bit rows end at K, 8-bit ones are padded with zeros)
                copy16(base + tok * sh.pitch + 16 * i, there ? row + k : x, there);
            }
        }
    } else {
        for (int tok = warp; tok < live; tok += W4_WARPS) {
            const X* row = x + (size_t)(tok0 + tok) * ldx;
            X* mine = reinterpret_cast<X*>(smem + tok * sh.pitch);
            for (int i = lane; i < count * 128; i += 32) mine[i] = first * 128 + i < K ? row[first * 128 + i] : static_cast<X>(0.f);
        }
    }
    if constexpr (BYTES) {
        const int here = count * GROUPS;
        for (int i = threadIdx.x; i < here * live; i += THREADS) {
            const int tok = i / here, gr = i - tok * here;
            const bool there = first * GROUPS + gr < all_groups;
            copy4(base + sh.scales + (gr * 8 * NB + tok) * 4, there ? xs + (size_t)(tok0 + tok) * all_groups + first * GROUPS + gr : xs, there);
        }
    }
    asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    float* sums = reinterpret_cast<float*>(smem + sh.sums);
    int rows[NB];                                        // (a token that is not there reads another's numbers: its sums are not written)
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) rows[nb] = min(8 * nb + g, live - 1) * sh.pitch + (128 * (from - first) + 8 * t) * (int)sizeof(X);
    const int scales0 = sh.scales + ((from - first) * GROUPS * 8 * NB + 2 * t) * 4, slots0 = sh.ring + warp * DEPTH * SLOT;
    int slot = slots0;
    unsigned long long acc[RT][NB][2] = {};              // [tile][eight tokens][row g, g + 8] of two tokens

    // a round's sums, over the warps of a tile and the CTAs of the cluster in order; every CTA writes a share
    auto write_round = [&](int round) {
        const float* at = sums + (splits > 1 ? round & 1 : 0) * 8 * NB * SUMS;
        const int rows_here = 16 * RT * at_once, n0 = (round * clusters + cluster) * rows_here;
        for (int i = rank * THREADS + threadIdx.x; i < live * rows_here / 4; i += splits * THREADS) {
            const int tok = i / (rows_here / 4), r = (i - tok * (rows_here / 4)) * 4;
            const float* p = at + tok * SUMS + r / (16 * RT) * ways * 16 * RT + r % (16 * RT);
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (splits == 1) {
#pragma unroll 4
                for (int k = 0; k < ways; ++k) {
                    const float4 f = *reinterpret_cast<const float4*>(p + 16 * RT * k);
                    v.x += f.x, v.y += f.y, v.z += f.z, v.w += f.w;
                }
            } else {
                const uint32_t here = (uint32_t)__cvta_generic_to_shared(p);
#pragma unroll 4                                        // (loads before sums: a peer's shared memory is far)
                for (int j = 0, c = 0, k = 0; j < splits * ways; ++j) {
                    uint32_t there;
                    float4 f;
                    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(here), "r"(c));
                    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(f.x), "=f"(f.y), "=f"(f.z), "=f"(f.w) : "r"(there + 64 * RT * k));
                    if (++k == ways) k = 0, ++c;
                    v.x += f.x, v.y += f.y, v.z += f.z, v.w += f.w;
                }
            }
            w4_write4(o, tok0 + tok, n0 + r, v);
        }
    };

    for (int round = 0; round < rounds; ++round) {
        if (tile_of(round) < tiles)
            for (int u = 0; u < to - from; ++u) {
                asm volatile("cp.async.wait_group %0;" ::"n"(DEPTH - 1) : "memory");
                __syncwarp();
                const uint8_t* here = smem + slot;
                uint32_t lo[RT][4], hi[RT][4];
                float sw[RT][GROUPS][2];
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    const uint4 wa = *reinterpret_cast<const uint4*>(here + r * W4_SLOT + 16 * lane), wb = *reinterpret_cast<const uint4*>(here + r * W4_SLOT + 512 + 16 * lane);
                    lo[r][0] = wa.x; lo[r][1] = wa.y; lo[r][2] = wb.x; lo[r][3] = wb.y;
                    hi[r][0] = wa.z; hi[r][1] = wa.w; hi[r][2] = wb.z; hi[r][3] = wb.w;
#pragma unroll
                    for (int p = 0; p < GROUPS; ++p) {
                        const uint32_t s2 = *reinterpret_cast<const uint32_t*>(here + r * W4_SLOT + 1024 + (8 * p + g) * 4);
                        sw[r][p][0] = __uint_as_float(s2 << 16); sw[r][p][1] = __uint_as_float(s2 & 0xffff0000u);
                        if (BYTES) { sw[r][p][0] *= 0.0625f; sw[r][p][1] *= 0.0625f; }    // the products hold 16 q
                    }
                }
                __syncwarp();                            // all have read the slot
                ask();
                slot = slot == slots0 + (DEPTH - 1) * SLOT ? slots0 : slot + SLOT;
                const uint8_t* numbers = smem + 128 * (int)sizeof(X) * u;
                const uint8_t* scales = smem + scales0 + GROUPS * 8 * NB * 4 * u;
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    const uint8_t* row = numbers + rows[nb];
                    if constexpr (BYTES) {
                        const int start[4] = {0x4b400000, 0x4b400000, 0x4b400000, 0x4b400000};
                        int c[RT][GROUPS][4];
#pragma unroll
                        for (int h = 0; h < 4; ++h) {
                            const uint2 x8 = *reinterpret_cast<const uint2*>(row + 32 * h);
#pragma unroll
                            for (int r = 0; r < RT; ++r) {
                                int (&part)[4] = c[r][h / QUARTERS];
                                quarter(part, h % QUARTERS ? part : start, lo[r][h], hi[r][h], x8);
                            }
                        }
#pragma unroll
                        for (int p = 0; p < GROUPS; ++p) {
                            const unsigned long long xa = *reinterpret_cast<const unsigned long long*>(scales + (p * 8 * NB + 8 * nb) * 4), less = two(-12582912.f, -12582912.f);
#pragma unroll
                            for (int r = 0; r < RT; ++r)
#pragma unroll
                                for (int e = 0; e < 2; ++e)
                                    acc[r][nb][e] = fma_two(add_two(two(__int_as_float(c[r][p][2 * e]), __int_as_float(c[r][p][2 * e + 1])), less),
                                                            mul_two(xa, two(sw[r][p][e], sw[r][p][e])), acc[r][nb][e]);
                        }
                    } else {
                        const float start[4] = {};
                        float c[RT][GROUPS][4];
#pragma unroll
                        for (int h = 0; h < 4; ++h) {
                            const uint4 x8 = *reinterpret_cast<const uint4*>(row + 64 * h);
#pragma unroll
                            for (int r = 0; r < RT; ++r) {
                                float (&part)[4] = c[r][h / QUARTERS];
                                quarter(part, h % QUARTERS ? part : start, lo[r][h], hi[r][h], x8);
                            }
                        }
#pragma unroll
                        for (int r = 0; r < RT; ++r)
#pragma unroll
                            for (int p = 0; p < GROUPS; ++p)
#pragma unroll
                                for (int e = 0; e < 2; ++e)
                                    acc[r][nb][e] = fma_two(two(c[r][p][2 * e], c[r][p][2 * e + 1]), two(sw[r][p][e], sw[r][p][e]), acc[r][nb][e]);
                    }
                }
            }
        if (splits == 1 && ways == 1) {                  // the warp's own tile: straight out, eight rows of a token at a time
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float a, c;
                        asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(c) : "l"(acc[r][nb][e]));
                        const int n = (tile_of(round) * RT + r) * 16 + g + 8 * e, tok = 8 * nb + 2 * t;
                        if (tok < live) w4_write(o, tok0 + tok, n, a);
                        if (tok + 1 < live) w4_write(o, tok0 + tok + 1, n, c);
                        acc[r][nb][e] = 0ull;
                    }
            continue;
        }
        if (splits > 1 && round > 0) {
            __syncwarp();
            asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
            write_round(round - 1);
        }
        if (splits == 1 && ways > 1 && round > 0) __syncthreads();              // the sums of the round before are read
        float* to_a = sums + ((splits > 1 ? round & 1 : 0) * 8 * NB + 2 * t) * SUMS + 16 * RT * warp + g;
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float a, c;
                    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(c) : "l"(acc[r][nb][e]));
                    to_a[8 * nb * SUMS + 16 * r + 8 * e] = a;
                    to_a[(8 * nb + 1) * SUMS + 16 * r + 8 * e] = c;
                    acc[r][nb][e] = 0ull;
                }
        if (splits > 1) {
            // two sets of sums in turn: who writes a set for the second time knows, by the barrier between, that all have read the first
            __syncwarp();                                // (the lanes wrote the round before in loops of different lengths)
            asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        } else {
            __syncthreads();
            write_round(round);
        }
    }
    if (splits > 1) {
        __syncwarp();
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        write_round(rounds - 1);
        // a CTA's shared memory stays until its peers have read it
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
}

// ---------------------------------------------------------------- launchers
// f(G as a constant)
template <typename F>
static void with_group(int G, F f) {
    if (G == 32) f(std::integral_constant<int, 32>());
    else if (G == 64) f(std::integral_constant<int, 64>());
    else f(std::integral_constant<int, 128>());
}
static dim3 place_grid(int T_, int Kp, int each) {
    const int units = Kp / each, across = units < 256 ? 256 / units : 1, rows = (T_ + across - 1) / across;
    return dim3((units + 255) / 256, rows < 65535 ? rows : 65535);
}

template <typename T>
static int launch_quantize_q8(const T* x, long long ldx, int8_t* q, float* s, int T_, int K, int G, cudaStream_t st) {
    const int Kp = padded(K, G);
    const bool vec = K % 4 == 0 && ldx % 4 == 0 && aligned(x, 4 * sizeof(T));
    with_group(G, [&](auto gc) {
        constexpr int GC = decltype(gc)::value;
        if (vec) rf_launch(quantize_q8_kernel<T, GC, true>, place_grid(T_, Kp, 4), dim3(256), 0, st, x, ldx, q, s, T_, K, Kp);
        else rf_launch(quantize_q8_kernel<T, GC, false>, place_grid(T_, Kp, 4), dim3(256), 0, st, x, ldx, q, s, T_, K, Kp);
    });
    RF_LAUNCH_CHECK();
    return 0;
}

template <typename T, int ACT>
static int launch_swiglu_q8(const T* gu, int8_t* q, float* s, int T_, int I, int G, cudaStream_t st) {
    const int Ip = padded(I, G);
    const bool vec = I % 2 == 0 && aligned(gu, 4 * sizeof(T));
    with_group(G, [&](auto gc) {
        constexpr int GC = decltype(gc)::value;
        if (vec) rf_launch(swiglu_q8_kernel<T, ACT, GC, true>, place_grid(T_, Ip, 4), dim3(256), 0, st, gu, q, s, T_, I, Ip);
        else rf_launch(swiglu_q8_kernel<T, ACT, GC, false>, place_grid(T_, Ip, 4), dim3(256), 0, st, gu, q, s, T_, I, Ip);
    });
    RF_LAUNCH_CHECK();
    return 0;
}

template <typename T>
static int launch_add_rmsnorm_q8(float* h, const void* pending, int kind, int n_pending, size_t pstride, const void* w, int w_is_f32, float eps,
                                 int8_t* q, float* s, const int* rows, int n_rows, int n_h, int H, int G, cudaStream_t st) {
    const int Hp = padded(H, G), quads = Hp / 4;
    if (quads > 8 * 1024) return RF_ERR_UNSUPPORTED;
    const bool vec = H % 4 == 0 && pstride % 4 == 0 && aligned(h, 16) && (kind == 0 || aligned(pending, kind == 1 ? 16 : 4 * sizeof(T)));
    int per = (quads + 1023) / 1024;
    per = per <= 1 ? 1 : per <= 2 ? 2 : 8;
    // Two quads a thread where there are rows for every SM and long ones: more of them at once (2,048 x 3,584 after a 16-bit update 22.3 -> 16.6 us,
    // four 17.9; 512 x 3,584 after four sums 11.0 -> 10.1).  Few or short rows want all the threads: 1 x 896 2.1 us, with two 3.0; 4,096 x 512
    // 10.2, 11.1.
    if (per == 1 && quads >= 384 && n_rows >= 2 * 148) per = 2;
    const int threads = ((quads + per - 1) / per + 31) / 32 * 32;
    with_group(G, [&](auto gc) {
        constexpr int GC = decltype(gc)::value;
        auto go = [&](auto kernel) {
            rf_launch(kernel, dim3(n_rows), dim3(threads), 0, st, h, pending, kind, n_pending, pstride, w, w_is_f32, eps, q, s, rows, n_h, H, Hp);
        };
        auto by_form = [&](auto v) {
            constexpr bool VEC = decltype(v)::value;
            if (per == 1) go(add_rmsnorm_q8_kernel<T, GC, 1, VEC>);
            else if (per == 2) go(add_rmsnorm_q8_kernel<T, GC, 2, VEC>);
            else go(add_rmsnorm_q8_kernel<T, GC, 8, VEC>);
        };
        if (vec) by_form(std::true_type());
        else by_form(std::false_type());
    });
    RF_LAUNCH_CHECK();
    return 0;
}

// f(group, rows, eights, tiles a warp) with the constants and types of a product's kernel; false: there is none (where four eights of 16-bit rows
// would pay, the tensor cores' kernel takes less)
template <typename F>
static bool with_product(int x_kind, int G, int eights, int pair, F f) {
    using One = std::integral_constant<int, 1>;
    using Two = std::integral_constant<int, 2>;
    using Four = std::integral_constant<int, 4>;
    if (!(eights == 1 && pair == 1) && !(eights == 2 && (pair == 1 || pair == 2)) && !(eights == 4 && (pair == 1 || pair == 2) && x_kind == 0)) return false;
    with_group(G, [&](auto gc) {
        const int8_t* bytes = nullptr;
        const __nv_bfloat16* wide = nullptr;
        auto few = [&](auto rows) {
            if (eights == 1) f(gc, rows, One(), One());
            else if (pair == 1) f(gc, rows, Two(), One());
            else f(gc, rows, Two(), Two());
        };
        if (x_kind != 0) few(wide);
        else if (eights < 4) few(bytes);
        else if (pair == 1) f(gc, bytes, Four(), One());
        else f(gc, bytes, Four(), Two());
    });
    return true;
}
template <int G, typename X, int NB, int RT>
static int set_shared() {                                // the kernel's limit of shared memory, once a device
    static PerDevice<bool> set;
    bool& done = set.here();
    if (done) return 0;
    const cudaError_t e = cudaFuncSetAttribute(w4_product_kernel<G, X, NB, RT>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
    done = e == cudaSuccess;
    return (int)e;
}
#define W4_MOST_SHARED (227 * 1024)

extern "C" {

// x [T, K] (rows ldx apart) -> q int8 [T, Kp], scales float32 [T, Kp / G]; Kp: K up to a multiple of 64 (128 if G is).
int rf_quantize_q8(int dtype, const void* x, long long ldx, void* q, void* scales, int T_, int K, int G, cudaStream_t st) {
    if (T_ < 0 || K <= 0 || bad_group(G)) return RF_ERR_BAD_ARG;
    if (T_ == 0) return 0;
    return dtype == 0 ? launch_quantize_q8((const float*)x, ldx, (int8_t*)q, (float*)scales, T_, K, G, st)
                      : launch_quantize_q8((const __nv_bfloat16*)x, ldx, (int8_t*)q, (float*)scales, T_, K, G, st);
}

int rf_dequantize_q8(int dtype, const void* q, const void* scales, void* y, int T_, int K, int G, cudaStream_t st) {
    if (T_ < 0 || K <= 0 || bad_group(G)) return RF_ERR_BAD_ARG;
    if (T_ == 0) return 0;
    const int Kp = padded(K, G);
    auto go = [&](auto kernel, auto* out, int each) { rf_launch(kernel, place_grid(T_, Kp, each), dim3(256), 0, st, (const int8_t*)q, (const float*)scales, out, T_, K, Kp, G); };
    const bool eights = K % 8 == 0 && aligned(y, 16);
    if (dtype == 0 && eights) go(dequantize_q8_kernel<float, 8>, (float*)y, 8);
    else if (dtype == 0) go(dequantize_q8_kernel<float, 4>, (float*)y, 4);
    else if (eights) go(dequantize_q8_kernel<__nv_bfloat16, 8>, (__nv_bfloat16*)y, 8);
    else go(dequantize_q8_kernel<__nv_bfloat16, 4>, (__nv_bfloat16*)y, 4);
    RF_LAUNCH_CHECK();
    return 0;
}

// act 0: silu, 1: relu, 2: gelu by tanh
int rf_swiglu_q8(int dtype, const void* gu, int act, void* q, void* scales, int T_, int I, int G, cudaStream_t st) {
    if (T_ < 0 || I <= 0 || bad_group(G) || act < 0 || act > 2) return RF_ERR_BAD_ARG;
    if (T_ == 0) return 0;
    auto go = [&](auto p) {
        int8_t* qq = (int8_t*)q;
        float* ss = (float*)scales;
        return act == 0 ? launch_swiglu_q8<std::remove_cv_t<std::remove_pointer_t<decltype(p)>>, 0>(p, qq, ss, T_, I, G, st)
             : act == 1 ? launch_swiglu_q8<std::remove_cv_t<std::remove_pointer_t<decltype(p)>>, 1>(p, qq, ss, T_, I, G, st)
                        : launch_swiglu_q8<std::remove_cv_t<std::remove_pointer_t<decltype(p)>>, 2>(p, qq, ss, T_, I, G, st);
    };
    return dtype == 0 ? go((const float*)gu) : go((const __nv_bfloat16*)gu);
}

int rf_add_rmsnorm_q8(int dtype, float* h, const void* pending, int kind, int n_pending, long long pstride, const void* w, int w_is_f32, float eps,
                      void* q, void* scales, const int* rows, int n_rows, int n_h, int H, int G, cudaStream_t st) {
    if (n_rows < 0 || n_h < 0 || H <= 0 || bad_group(G) || kind < 0 || kind > 2 || n_pending < 0) return RF_ERR_BAD_ARG;
    if (n_rows == 0) return 0;
    if (n_h == 0) return RF_ERR_BAD_ARG;
    return dtype == 0 ? launch_add_rmsnorm_q8<float>(h, pending, kind, n_pending, (size_t)pstride, w, w_is_f32, eps, (int8_t*)q, (float*)scales, rows, n_rows, n_h, H, G, st)
                      : launch_add_rmsnorm_q8<__nv_bfloat16>(h, pending, kind, n_pending, (size_t)pstride, w, w_is_f32, eps, (int8_t*)q, (float*)scales, rows, n_rows, n_h, H, G, st);
}

// weight [N, K] (rows ldw apart) -> packed, scales (the layout above)
int rf_quantize_w4(int dtype, const void* weight, long long ldw, void* packed, void* scales, int N, int K, int G, cudaStream_t st) {
    if (N <= 0 || K <= 0 || bad_group(G)) return RF_ERR_BAD_ARG;
    const int Kp = padded(K, G);
    const long long units = (long long)((N + 15) / 16) * (Kp / (G == 128 ? 128 : 64));
    if ((units + 7) / 8 > 0x7fffffffll) return RF_ERR_UNSUPPORTED;
    with_group(G, [&](auto gc) {
        constexpr int GC = decltype(gc)::value;
        const dim3 grid((unsigned)((units + 7) / 8));
        if (dtype == 0) quantize_w4_kernel<float, GC><<<grid, 256, 0, st>>>((const float*)weight, ldw, (uint4*)packed, (__nv_bfloat16*)scales, N, K, Kp);
        else quantize_w4_kernel<__nv_bfloat16, GC><<<grid, 256, 0, st>>>((const __nv_bfloat16*)weight, ldw, (uint4*)packed, (__nv_bfloat16*)scales, N, K, Kp);
    });
    weights_made_kernel<<<1, 32, 0, st>>>();
    RF_LAUNCH_CHECK();
    return 0;
}

int rf_dequantize_w4(int dtype, const void* packed, const void* scales, void* out, int N, int K, int lo, int hi, int G, cudaStream_t st) {
    if (N <= 0 || K <= 0 || bad_group(G) || lo < 0 || lo % 64 || hi <= lo || hi > K || !aligned(out, 16)) return RF_ERR_BAD_ARG;
    const int Kp = padded(K, G);
    const long long units = (long long)((N + 15) / 16) * ((hi - lo + 63) / 64);
    if ((units + 7) / 8 > 0x7fffffffll) return RF_ERR_UNSUPPORTED;
    with_group(G, [&](auto gc) {
        constexpr int GC = decltype(gc)::value;
        const dim3 grid((unsigned)((units + 7) / 8));
        if (dtype == 0) rf_launch(dequantize_w4_kernel<float, GC>, grid, dim3(256), 0, st, (const uint4*)packed, (const __nv_bfloat16*)scales, (float*)out, N, Kp, lo, hi);
        else rf_launch(dequantize_w4_kernel<__nv_bfloat16, GC>, grid, dim3(256), 0, st, (const uint4*)packed, (const __nv_bfloat16*)scales, (__nv_bfloat16*)out, N, Kp, lo, hi);
    });
    weights_made_kernel<<<1, 32, 0, st>>>();
    RF_LAUNCH_CHECK();
    return 0;
}

// Lets products that follow read weights that the stream's last kernels have made (see weights_made_kernel).
int rf_weights_made(cudaStream_t st) {
    weights_made_kernel<<<1, 32, 0, st>>>();
    RF_LAUNCH_CHECK();
    return 0;
}

// Bytes of shared memory that a product's block takes with `eights` eights of tokens, `pair` tiles of 16 rows a warp, `ways` warps a tile, a
// share of the columns in `splits` and `clusters` clusters.
int rf_gemm_w4_shared(int x_kind, int M, int N, int K, int G, int eights, int pair, int ways, int splits, int clusters) {
    return w4_shared((padded(K, G) / 64 + 1) / 2, w4_rounds(N, pair, ways, clusters), ways, splits, G, x_kind == 0 ? 1 : 2, M, eights, pair).bytes;
}

// Clusters of `splits` blocks, each with an SM of its own, that run at once on the current device (< 0: an error).
int rf_gemm_w4_clusters(int splits) {
    if (splits < 1 || splits > 8) return RF_ERR_BAD_ARG;
    if (const int e = set_shared<128, int8_t, 1, 1>()) return -e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(splits);
    cfg.blockDim = dim3(32 * W4_WARPS);
    cfg.dynamicSmemBytes = W4_MOST_SHARED;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = splits; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    const cudaError_t e = cudaOccupancyMaxActiveClusters(&n, w4_product_kernel<128, int8_t, 1, 1>, &cfg);
    return e == cudaSuccess ? n : -(int)e;
}

// out = x w^T (+ bias): x_kind 0: 8-bit rows (x int8 [M, Kp], xs float32 [M, Kp / G]), 1: bfloat16 rows [M, K], ldx apart; out as W4Out
// has it.  eights: eights of tokens a block (1, 2; 8-bit rows 4 too); pair: tiles of 16 rows a warp (1; 2 from two eights on); ways: warps a tile
// (a power of two up to 16); splits: CTAs of a cluster that share out the columns (1 .. 8); clusters: of each share of tokens.
int rf_gemm_w4(int x_kind, const void* x, const void* xs, long long ldx, const void* packed, const void* scales, const void* bias, int bias_is_f32,
               void* out, int out_is_f32, int add, int eights, int pair, int ways, int splits, int clusters, int M, int N, int K, int G, cudaStream_t st) {
    if (M <= 0 || N <= 0 || K <= 0 || bad_group(G) || (add && !out_is_f32)) return RF_ERR_BAD_ARG;
    if ((x_kind == 0 && (!aligned(x, 16) || ldx % 16)) || !aligned(packed, 16) || !aligned(scales, 16)) return RF_ERR_BAD_ARG;
    if (splits < 1 || splits > 8 || clusters < 1 || ways < 1 || ways > W4_WARPS || (ways & (ways - 1)) || eights < 1) return RF_ERR_BAD_ARG;
    const int whole = x_kind == 0 || (K % 8 == 0 && ldx % 8 == 0 && aligned(x, 16));
    const int blocks = padded(K, G) / 64, smem = rf_gemm_w4_shared(x_kind, M, N, K, G, eights, pair < 1 ? 1 : pair, ways, splits, clusters);
    const long long y = (M + 8ll * eights - 1) / (8 * eights);
    if (smem > W4_MOST_SHARED || y > 65535 || (long long)clusters * splits > 0x7fffffffll) return RF_ERR_UNSUPPORTED;
    const W4Out o = w4_out(out, bias, bias_is_f32, out_is_f32, add, M, N);
    int bad = 0;
    const bool known = with_product(x_kind, G, eights, pair, [&](auto gc, auto rows, auto nb, auto rt) {
        using X = std::remove_cv_t<std::remove_pointer_t<decltype(rows)>>;
        constexpr int GC = decltype(gc)::value, NB = decltype(nb)::value, RT = decltype(rt)::value;
        bad = set_shared<GC, X, NB, RT>();
        if (bad) return;
        const dim3 grid(clusters * splits, (unsigned)y), block(32 * W4_WARPS);
        auto go = [&](auto... args) {
            if (splits > 1) rf_launch_cluster(w4_product_kernel<GC, X, NB, RT>, grid, block, smem, st, splits, args...);
            else rf_launch(w4_product_kernel<GC, X, NB, RT>, grid, block, smem, st, args...);
        };
        go((const uint4*)packed, (const uint32_t*)scales, (const X*)x, (const float*)xs, ldx, whole, K, blocks, ways, splits, o);
    });
    if (!known) return RF_ERR_BAD_ARG;
    if (bad) return bad;
    RF_LAUNCH_CHECK();
    return 0;
}

}  // extern "C"
