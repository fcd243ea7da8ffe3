// Products of bfloat16 rows with 4-bit weights on the 5th-generation tensor cores, from 17 tokens on.
//
// Weights are the accumulator's rows, tokens its columns.  128 rows of weights go through shared memory a stage at a time: eight warps have a
// tile of 16 rows each as it is stored, in registers, asked for AHEAD stages before (and before the wait for the kernel before); they widen
// it to bfloat16 numbers, scale and all (exactly, with scales of five significant bits; others are rounded), and write it where the MMA
// reads it.  Two groups of eight warps do every second stage each.  The tokens' numbers come by TMA into a ring of their own.  Long rows are
// shared out to the CTAs of a cluster, which add up their sums through shared memory in the order of their ranks.
//
// The tensor cores cut what an addition loses instead of rounding it, and what is cut adds up (1,999 x 3,584 x 18,944 against 64 bits: one sum
// 1.1e-5 off, pieces of 6,315 columns 2.6e-6).  For 32-bit results a sum runs over W4T_PIECE columns at most: the widening warps add it to a
// second one beside it, rounded, while the next piece goes into another accumulator (tiles of 256 tokens: into the same one, after a wait).
//
// Every wait on an mbarrier is bounded (2 s): status word 13.
#include <type_traits>
#include "quantized.cuh"
#include "tcgen05_common.cuh"

#define W4T_THREADS (32 * 18)                            // the tokens' producer, the MMA issuer, sixteen widening warps (which write the result)
#define W4T_PIECE 2048                                   // columns of one sum where the result is 32-bit
#define W4T_PITCH (128 + 4)                              // of the sums that a cluster exchanges, [token][row]
#define W4T_MOST_SHARED (226 * 1024)                     // (the abort flag has a place of its own)

template <int BN, int G>
struct TcShape {
    static constexpr int BLOCKS = BN <= 64 ? 2 : 1;      // blocks of 64 columns a stage: what a stage costs beside its work, twice as rarely
    static constexpr int A = BLOCKS * 128 * 128, B = BLOCKS * BN * 128;
    static constexpr int STAGES = 4, ROWS = BN == 128 ? 8 : 4;          // places of weights, of tokens' numbers
    static constexpr int TURN = STAGES / 2;              // a warp's stages until it is back at the same place (a group sees all phases of it)
    static constexpr int AHEAD = BLOCKS == 2 && G == 32 ? 2 : 4;        // stages of its own that a warp has asked for (more scales leave room for fewer)
    static constexpr int PIECE = W4T_PIECE / 64 / BLOCKS;                               // stages of a piece
    static constexpr int BUFS = BN <= 128 ? 2 : 1, TMEM = BN == 256 ? 512 : 4 * BN;     // accumulators; with them, behind, the pieces' sum
    static constexpr int SHARE = BN / 4 < 16 ? 16 : BN / 4;             // a widening warp's part of the sums: 32 rows, so many tokens
    static_assert(PIECE % 8 == 0 && PIECE / 2 % AHEAD == 0 && AHEAD % TURN == 0, "pieces end between turns");
    static constexpr int RINGS = STAGES * A + ROWS * B, BYTES = RINGS + 1024 + 256;     // (alignment, barriers)
    static_assert(RINGS >= BN * W4T_PITCH * 4, "the rings' place holds the sums");
    static_assert(BYTES <= W4T_MOST_SHARED && 8 % ROWS == 0 && 8 % STAGES == 0, "eight stages on, every ring is back where it was (one of eight with the parity turned)");
};

// Bounded wait as mbar_wait, asleep between looks: what waits here waits long, and the widening warps need the issue slots.
__device__ __noinline__ bool wait_asleep(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
    const unsigned long long t0 = global_ns();
    for (;;) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok) : "r"(bar), "r"(parity), "r"(20000u) : "memory");
        if (ok) return true;
        if (*abort_flag) return false;
        if (global_ns() - t0 > TC_WAIT_LIMIT_NS) { *abort_flag = 1; return false; }
    }
}
__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
    return mbar_try_wait(bar, parity) || wait_asleep(bar, parity, abort_flag);
}

// Two halves of bytes, 16 bits apart, as bfloat16 numbers times a scale.
__device__ __forceinline__ uint32_t widened(uint32_t w, __nv_bfloat162 s) {
    uint32_t v = (w & 0x000f000fu) ^ 0x43084308u;        // 128 + (q + 8)
    const __nv_bfloat162 r = __hmul2(__hadd2(*reinterpret_cast<__nv_bfloat162*>(&v), __float2bfloat162_rn(-136.f)), s);
    return *reinterpret_cast<const uint32_t*>(&r);
}
// A word's eight columns into 16 bytes of shared memory; with the middle bytes swapped, neighbours are 16 bits apart.
__device__ __forceinline__ void four_pairs(uint32_t at, uint32_t word, uint32_t scale_twice) {
    const uint32_t w = __byte_perm(word, 0, 0x3120);
    const __nv_bfloat162 s = *reinterpret_cast<const __nv_bfloat162*>(&scale_twice);
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};"
                 ::"r"(at), "r"(widened(w, s)), "r"(widened(w >> 8, s)), "r"(widened(w >> 4, s)), "r"(widened(w >> 12, s)) : "memory");
}

// A widening warp's share of a piece's sum added to the sum of those before.
template <int BN, int G>
__device__ __noinline__ bool add_piece(uint32_t tmem, uint32_t sum_full, int piece, volatile int* abort_flag) {
    using S = TcShape<BN, G>;
    const int buf = piece % S::BUFS, warp = threadIdx.x >> 5, share = (warp - 2) / 4 * S::SHARE;
    if (!__all_sync(0xffffffffu, wait_for(sum_full + 8 * buf, piece / S::BUFS & 1, abort_flag))) return false;
    tcgen05_fence_after();
    if (share < BN) {
        const uint32_t rows = tmem + ((uint32_t)((warp & 3) * 32) << 16) + share;
#pragma unroll 1
        for (int c = 0; c < S::SHARE; c += 16) {
            uint32_t a[16], b[16];
            tcgen05_ld16(rows + buf * BN + c, a);
            if (piece > 0) tcgen05_ld16(rows + S::BUFS * BN + c, b);
            tcgen05_wait_ld();
            if (piece > 0) {
#pragma unroll
                for (int j = 0; j < 16; ++j) a[j] = __float_as_uint(__uint_as_float(a[j]) + __uint_as_float(b[j]));
            }
            tcgen05_st16(rows + S::BUFS * BN + c, a);
        }
        tcgen05_wait_st();
    }
    tcgen05_fence_before();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) at_arrive(sum_full + 8 * (S::BUFS + buf));
    return true;
}

// 32 rows of sixteen tokens (from c on) of the result: the last piece's sum and that of those before, into `sums` ([token][row]) or, without,
// straight out.  (Functions of their own keep these parts' registers out of the loop over the weights: written there, 64 x 37,888 x 3,584 took
// 51 us, not 36.)
__device__ __noinline__ void write_16(uint32_t last_sum, uint32_t sum_before, bool any, bool more, float* sums, int row0, int c, int tok0, int live, W4Out o) {
    uint32_t r[16], before[16];
    float old[16];
    if (any) tcgen05_ld16(last_sum + c, r);
    if (more) tcgen05_ld16(sum_before + c, before);
    const int at_row = 32 * (threadIdx.x >> 5 & 3) + (threadIdx.x & 31), row = row0 + at_row;
    const bool there = row < o.N;
    const size_t to = (size_t)(tok0 + c) * o.N + row;
    const float bias = there && o.bias != nullptr ? load_vec(o.bias, o.bias_is_f32, row) : 0.f;
    if (sums == nullptr && o.add) {                      // (all at once: a load after every store would wait for it)
#pragma unroll
        for (int j = 0; j < 16; ++j) old[j] = there && c + j < live ? reinterpret_cast<const float*>(o.out)[to + (size_t)j * o.N] : 0.f;
    }
    tcgen05_wait_ld();
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        const float v = any ? __uint_as_float(r[j]) + (more ? __uint_as_float(before[j]) : 0.f) : 0.f;
        if (sums != nullptr) sums[(c + j) * W4T_PITCH + at_row] = v;
        else if (there && c + j < live) {
            if (o.add) reinterpret_cast<float*>(o.out)[to + (size_t)j * o.N] = v + bias + old[j];
            else if (o.is_f32) reinterpret_cast<float*>(o.out)[to + (size_t)j * o.N] = v + bias;
            else reinterpret_cast<__nv_bfloat16*>(o.out)[to + (size_t)j * o.N] = __float2bfloat16_rn(v + bias);
        }
    }
}

template <int BN, int G>
__global__ void __launch_bounds__(W4T_THREADS, 1) w4_tc_kernel(const __grid_constant__ CUtensorMap map_x, const uint4* __restrict__ w0, const uint32_t* __restrict__ w1,
                                                               int blocks, int splits, bool pieces, int* status, W4Out o) {
    using S = TcShape<BN, G>;
    constexpr int SCALES = S::BLOCKS * 64 > G ? S::BLOCKS * 64 / G : 1;                 // groups that a stage touches
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::RINGS);                      // weights' places full, empty, tokens' full, empty, sums full, added
    constexpr int FULL = 0, EMPTY = S::STAGES, ROWS_FULL = 2 * S::STAGES, ROWS_EMPTY = ROWS_FULL + S::ROWS, SUMS = ROWS_EMPTY + S::ROWS, ADDED = SUMS + S::BUFS;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + ADDED + S::BUFS);
    __shared__ int abort_flag;
    pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = blockIdx.x % splits, row0 = blockIdx.x / splits * 128, tok0 = blockIdx.y * BN, live = min(BN, o.M - tok0);
    const int all = (blocks + S::BLOCKS - 1) / S::BLOCKS, from = (int)((long long)all * rank / splits);
    const int n = (int)((long long)all * (rank + 1) / splits) - from;
    const int tiles = (o.N + 15) / 16, all_groups = blocks * 64 / G;
    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int i = 0; i < S::STAGES; ++i) {
            mbar_init(smem_u32(&bars[FULL + i]), 8);     // eight widening warps
            mbar_init(smem_u32(&bars[EMPTY + i]), 1);
        }
        for (int i = 0; i < 2 * S::ROWS + S::BUFS; ++i) mbar_init(smem_u32(&bars[ROWS_FULL + i]), 1);
        for (int i = 0; i < S::BUFS; ++i) mbar_init(smem_u32(&bars[ADDED + i]), 16);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
    }
    if (warp == 1) {
        tcgen05_alloc(smem_u32(tmem_slot), S::TMEM);
        tcgen05_relinquish();
    }
    // the widening warps' weights: stages phase, phase + 2, ... of a tile of 16 rows, AHEAD of them in registers before anything is waited for
    const int wide = warp - 2, tile = min(row0 / 16 + (wide & 7), tiles - 1), phase = wide >> 3;        // (rows that are not there: some others)
    const int block0 = (from + phase) * S::BLOCKS, stages = wide >= 0 ? (n - phase + 1) / 2 : 0;
    const uint4* next_w = w0 + ((size_t)tile * blocks + block0) * 32 + lane;
    const uint32_t* next_s = w1 + ((size_t)tile * all_groups + block0 * 64 / G) * 8 + (lane >> 2);
    uint4 w[S::AHEAD][S::BLOCKS];
    uint32_t sc[S::AHEAD][SCALES];
    int asked = 0;
    auto ask = [&](int into) {
        if (asked < stages) {
            // (the last stage's second block may not be there)
            const bool second = S::BLOCKS == 2 && (asked + 1 < stages || block0 + 2 * S::BLOCKS * (stages - 1) + 1 < blocks);
            w[into][0] = next_w[0];
            if constexpr (S::BLOCKS == 2) w[into][1] = second ? next_w[32] : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
            for (int p = 0; p < SCALES; ++p) sc[into][p] = S::BLOCKS == 1 || second || p * G < 64 ? next_s[8 * p] : 0u;
            next_w += 2 * S::BLOCKS * 32;                // (two stages on are whole groups on)
            next_s += 2 * S::BLOCKS * 64 / G * 8;
            ++asked;
        }
    };
#pragma unroll
    for (int i = 0; i < S::AHEAD; ++i) ask(i);
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem = *tmem_slot;

    const int last = pieces && n > 0 ? (n - 1) / S::PIECE : 0;           // the piece that the result is read from, together with the sum of those before
    const uint32_t sum_full = smem_u32(&bars[SUMS]), added = smem_u32(&bars[ADDED]);
    bool ok = true;
    if (warp == 0) {
        // ---------------- the tokens' numbers
        if (lane == 0) {
            pdl_wait();
            const uint32_t full = smem_u32(&bars[ROWS_FULL]), empty = smem_u32(&bars[ROWS_EMPTY]), to = smem_u32(smem) + S::STAGES * S::A;
            for (int i = 0; i < n && ok; i += 8) {
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    if (i + u >= n) break;
                    const int at = u % S::ROWS;
                    if (i > 0 || u >= S::ROWS) ok = wait_for(empty + 8 * at, ((S::ROWS == 8 ? i / 8 : u / S::ROWS) & 1) ^ 1, &abort_flag);
                    if (!ok) break;
                    mbar_expect_tx(full + 8 * at, S::B);
#pragma unroll
                    for (int b = 0; b < S::BLOCKS; ++b)
                        tma_load_2d(to + at * S::B + b * BN * 128, &map_x, ((from + i + u) * S::BLOCKS + b) * 64, tok0, full + 8 * at);
                }
            }
        }
    } else if (warp == 1) {
        // ---------------- the products
        // Eight stages a turn, after which every ring is back where it was: places, parities and descriptors are constants.  (With remainders and
        // addresses formed anew this one thread, not the tensor cores, was the limit.)
        if (elect_one()) {
            const uint32_t full = smem_u32(&bars[FULL]), empty = smem_u32(&bars[EMPTY]), rows_full = smem_u32(&bars[ROWS_FULL]), rows_empty = smem_u32(&bars[ROWS_EMPTY]);
            const uint64_t da0 = make_smem_desc(smem_u32(smem)), db0 = make_smem_desc(smem_u32(smem) + S::STAGES * S::A);
            uint32_t sum = tmem;
            bool starts = true;
            for (int i = 0; i < n && ok; i += 8, starts = false) {
                if (pieces && i > 0 && i % S::PIECE == 0) {
                    const int piece = i / S::PIECE, buf = piece % S::BUFS;
                    tcgen05_commit(sum_full + 8 * ((piece - 1) % S::BUFS));
                    if (piece >= S::BUFS) ok = wait_for(added + 8 * buf, piece / S::BUFS - 1 & 1, &abort_flag);
                    if (!ok) break;
                    tcgen05_fence_after();
                    sum = tmem + buf * BN;
                    starts = true;
                }
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    if (i + u >= n) break;
                    const int a = u % S::STAGES, r = u % S::ROWS;
                    ok = wait_for(rows_full + 8 * r, (S::ROWS == 8 ? i / 8 : u / S::ROWS) & 1, &abort_flag) && wait_for(full + 8 * a, u / S::STAGES & 1, &abort_flag);
                    if (!ok) break;
                    tcgen05_fence_after();
#pragma unroll
                    for (int k = 0; k < 4 * S::BLOCKS; ++k) {           // 16 columns
                        const uint64_t da = da0 + (a * S::A + k / 4 * 128 * 128) / 16 + 2 * (k % 4), db = db0 + (r * S::B + k / 4 * BN * 128) / 16 + 2 * (k % 4);
                        tcgen05_mma_bf16(sum, da, db, make_idesc(BN), u || k || !starts ? 1u : 0u);
                    }
                    tcgen05_commit(empty + 8 * a);
                    tcgen05_commit(rows_empty + 8 * r);
                }
            }
            tcgen05_commit(sum_full + 8 * (last % S::BUFS));
        }
    } else {
        // ---------------- the weights
        const int g = lane >> 2, t = lane & 3;
        const bool odd = g & 1;
        // where this lane's 16 bytes of a row's half go (rows of 128 bytes, pieces swapped by row % 8 = g): by the row's parity the other half
        // first, so that two rows' pieces meet all banks
        uint32_t place[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) place[j] = smem_u32(smem) + phase * S::A + (16 * (wide & 7) + g) * 128 + (((4 * (odd ^ j) + t) ^ g) * 16);
        const uint32_t full = smem_u32(&bars[FULL + phase]), empty = smem_u32(&bars[EMPTY + phase]);
        int summed = 0;
        uint32_t parity = 1;
        for (int done = 0; done < stages && ok;) {
#pragma unroll
            for (int u = 0; u < S::AHEAD; ++u, ++done) {
                if (done >= stages) break;
                const int at = u % S::TURN * 2;
                // (a piece is added once the next one's first stages are on their way)
                if (u == S::TURN % S::AHEAD && (done - S::TURN) / (S::PIECE / 2) > summed && summed < last) {
                    ok = add_piece<BN, G>(tmem, smem_u32(&bars[SUMS]), summed, &abort_flag);
                    if (!ok) break;
                    ++summed;
                }
                if (done >= S::TURN) {
                    ok = wait_for(empty + 8 * at, parity, &abort_flag);
                    if (!ok) break;
                }
#pragma unroll
                for (int b = 0; b < S::BLOCKS; ++b) {
                    const uint4 v = w[u][b];
                    const uint32_t lo[2] = {odd ? v.y : v.x, odd ? v.x : v.y}, hi[2] = {odd ? v.w : v.z, odd ? v.z : v.w};
                    const uint32_t to = at * S::A + b * 128 * 128;
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const uint32_t s2 = G == 32 ? (odd ^ j ? sc[u][2 * b + 1] : sc[u][2 * b]) : sc[u][G == 64 ? b : 0];
                        four_pairs(place[j] + to, lo[j], __byte_perm(s2, 0, 0x1010));
                        four_pairs(place[j] + to + 8 * 128, hi[j], __byte_perm(s2, 0, 0x3232));
                    }
                }
                ask(u);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) at_arrive(full + 8 * at);
                if (u % S::TURN == S::TURN - 1) parity ^= 1;
            }
        }
        for (; ok && summed < last; ++summed) ok = add_piece<BN, G>(tmem, smem_u32(&bars[SUMS]), summed, &abort_flag);
    }
    pdl_wait();                                          // (whoever writes from here on has waited)
    // ---------------- the result: a warp has the same share as of the pieces; a cluster's go through the rings' place, one CTA's straight out
    const int share = (warp - 2) / 4 * S::SHARE;
    const bool writes = warp >= 2 && share < BN;
    if (writes && n > 0) {
        ok = wait_for(sum_full + 8 * (last % S::BUFS), last / S::BUFS & 1, &abort_flag) && ok;
        tcgen05_fence_after();
    }
    ok = __all_sync(0xffffffffu, ok);
    if (splits > 1) __syncthreads();                     // (the sums are there: every product has read the rings)
    if (writes && ok) {
        const uint32_t rows = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
#pragma unroll 1
        for (int c = share; c < share + S::SHARE; c += 16)
            write_16(rows + last % S::BUFS * BN, rows + S::BUFS * BN, n > 0, last > 0, splits > 1 ? reinterpret_cast<float*>(smem) : nullptr, row0, c, tok0, live, o);
    }
    if (splits > 1) {
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        for (int i = rank * W4T_THREADS + threadIdx.x; i < live * 32; i += splits * W4T_THREADS) {
            const int tok = i / 32, r = i % 32 * 4;
            const uint32_t here = smem_u32(smem) + (tok * W4T_PITCH + r) * 4;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
            for (int c = 0; c < splits; ++c) {
                uint32_t there;
                float4 f;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(here), "r"(c));
                asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(f.x), "=f"(f.y), "=f"(f.z), "=f"(f.w) : "r"(there));
                v.x += f.x, v.y += f.y, v.z += f.z, v.w += f.w;
            }
            if (!abort_flag) w4_write4(o, tok0 + tok, row0 + r, v);
        }
        // a CTA's shared memory stays until its peers have read it
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
    tcgen05_fence_before();
    __syncthreads();
    if (warp == 1) {
        tcgen05_fence_after();
        tcgen05_dealloc(tmem, S::TMEM);
    }
    if (threadIdx.x == 0 && abort_flag && status) atomicExch(status, 13);
}

// f(tokens of a tile, group) as constants; false where there is no such kernel
template <typename F>
static bool with_tc(int bn, int G, F f) {
    auto by_group = [&](auto b) {
        if (G == 32) f(b, std::integral_constant<int, 32>());
        else if (G == 64) f(b, std::integral_constant<int, 64>());
        else f(b, std::integral_constant<int, 128>());
    };
    if (bn == 32) by_group(std::integral_constant<int, 32>());
    else if (bn == 64) by_group(std::integral_constant<int, 64>());
    else if (bn == 128) by_group(std::integral_constant<int, 128>());
    else if (bn == 256) by_group(std::integral_constant<int, 256>());
    else return false;
    return true;
}

extern "C" {

// out = x w^T (+ bias): x bfloat16 [M, K], rows ldx apart, whole 16 bytes on 16-byte boundaries; out as W4Out has it.  bn: tokens of a tile (32, 64,
// 128, 256); splits: CTAs of a cluster that share out the columns (1 .. 8).
int rf_gemm_w4_tc(const void* x, long long ldx, const void* packed, const void* scales, const void* bias, int bias_is_f32, void* out, int out_is_f32, int add,
                  int bn, int splits, int M, int N, int K, int G, int* status, cudaStream_t st) {
    if (M <= 0 || N <= 0 || K <= 0 || bad_group(G) || (add && !out_is_f32) || splits < 1 || splits > 8 || bn < 1) return RF_ERR_BAD_ARG;
    if (!aligned(packed, 16) || !aligned(scales, 16) || ldx < K || ldx > 0x7fffffff) return RF_ERR_BAD_ARG;
    const int blocks = padded(K, G) / 64;
    const long long x_blocks = (long long)((N + 127) / 128) * splits, y = (M + (long long)bn - 1) / bn;
    if (x_blocks > 0x7fffffffll || y > 65535) return RF_ERR_UNSUPPORTED;
    CUtensorMap map;
    if (const int e = make_map(&map, x, M, K, ldx, bn)) return e;
    const W4Out o = w4_out(out, bias, bias_is_f32, out_is_f32, add, M, N);
    int bad = 0;
    const bool known = with_tc(bn, G, [&](auto b, auto g) {
        constexpr int BN = decltype(b)::value, GC = decltype(g)::value;
        static PerDevice<bool> set;
        bool& done = set.here();
        if (!done) {
            const cudaError_t e = cudaFuncSetAttribute(w4_tc_kernel<BN, GC>, cudaFuncAttributeMaxDynamicSharedMemorySize, TcShape<BN, GC>::BYTES);
            if (e != cudaSuccess) { bad = (int)e; return; }
            done = true;
        }
        const dim3 grid((unsigned)x_blocks, (unsigned)y), block(W4T_THREADS);
        auto go = [&](auto... args) {
            if (splits > 1) rf_launch_cluster(w4_tc_kernel<BN, GC>, grid, block, TcShape<BN, GC>::BYTES, st, splits, args...);
            else rf_launch(w4_tc_kernel<BN, GC>, grid, block, TcShape<BN, GC>::BYTES, st, args...);
        };
        go(map, (const uint4*)packed, (const uint32_t*)scales, blocks, splits, out_is_f32 != 0, status, o);
    });
    if (!known) return RF_ERR_BAD_ARG;
    if (bad) return bad;
    RF_LAUNCH_CHECK();
    return 0;
}

}  // extern "C"
