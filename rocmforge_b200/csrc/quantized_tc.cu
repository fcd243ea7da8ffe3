// Products with 4-bit weights on the 5th-generation tensor cores, for more tokens than mma.sync serves at the rate of memory.
//
// Weights are the accumulator's rows, tokens its columns.  128 rows of weights go through shared memory a stage at a time: eight warps fetch
// their tile of 16 rows as it is stored (asynchronous copies into a ring of their own, far ahead, and before the wait for the kernel
// before), widen it and write it where the MMA reads it; the tokens' numbers come by TMA.  A stage is 128 bytes of a row:
//   16-bit rows: 64 columns; the weights become bfloat16 numbers, scale and all (exactly, with scales of five significant bits; others are
//     rounded), and the whole product is one accumulator's.  Two groups of eight warps widen every second stage each.
//   8-bit rows: 128 columns; the weights become 16 q as signed bytes and a group's sum is exact in whole numbers, in an accumulator of its own,
//     which eight more warps read, scale by both scales and add to their 32-bit sums while the next groups are multiplied.
// Long rows are shared out to the CTAs of a cluster, which add up their sums through shared memory in the order of their ranks.
//
// Every wait on an mbarrier is bounded (2 s): status word 13.
#include <type_traits>
#include "quantized.cuh"
#include "tcgen05_common.cuh"

#define W4T_THREADS (32 * 18)                            // the tokens' producer, the MMA issuer, eight widening warps, eight adding warps
#define W4T_PITCH (128 + 4)                              // of the sums that a cluster exchanges, [token][row]

template <int BN, bool BYTES, int G>
struct TcShape {
    static constexpr int A = 128 * 128, B = BN * 128;
    static constexpr int WIDENS = BYTES ? 1 : 2;         // groups of widening warps: a group must see every second phase of a stage's barriers, or all
    static constexpr int STAGES = 4, ROWS = BYTES && BN == 128 ? 4 : 8;                // places of weights and, further ahead, of tokens' numbers
    static constexpr int RINGS = STAGES * A + ROWS * B;
    static constexpr int BLOCKS = BYTES ? 2 : 1;         // blocks of 64 columns a stage
    static constexpr int PARTS = BYTES ? 128 / G : 1;    // accumulators a stage
    static constexpr int BUFS = BYTES ? (BN <= 64 ? 4 : 2) : 1;
    static constexpr int TMEM = BUFS * BN < 32 ? 32 : BUFS * BN;
    static constexpr int SCALES = BYTES ? 0 : (G == 32 ? 2 : 1);        // groups of a stage whose scales the weights take
    static constexpr int TURN = STAGES / WIDENS;         // a warp's stages until it is back at the same place
    static constexpr int AHEAD = (BYTES ? 2 : 4) / TURN * TURN < TURN ? TURN : (BYTES ? 2 : 4) / TURN * TURN;      // its stages whose weights it has asked for
    static constexpr int FIXED = RINGS + 1024 + 512;           // (alignment, barriers)
    static_assert(RINGS >= BN * W4T_PITCH * 4, "the stages' place holds the sums");
    static_assert(STAGES % WIDENS == 0, "one parity bit tells two phases apart, not three");
    static_assert(8 % ROWS == 0 && 8 % STAGES == 0 && 8 * PARTS % (2 * BUFS) == 0, "eight stages on, every ring is back where it was");
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

template <int BN, bool BYTES>
__device__ __forceinline__ void mma_step(uint32_t d, uint64_t a, uint64_t b, uint32_t accumulate) {
    if constexpr (BYTES) {
        constexpr uint32_t idesc = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(BN >> 3) << 17) | (8u << 24);       // signed bytes, 32-bit whole sums
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
    } else {
        tcgen05_mma_bf16(d, a, b, make_idesc(BN), accumulate);
    }
}

__device__ __forceinline__ void to_shared8(uint32_t at, uint32_t a, uint32_t b) {
    asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(at), "r"(a), "r"(b) : "memory");
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

template <int BN, bool BYTES, int G>
__global__ void __launch_bounds__(W4T_THREADS, 1) w4_tc_kernel(const __grid_constant__ CUtensorMap map_x, const uint4* __restrict__ w0, const uint32_t* __restrict__ w1,
                                                               const float* xs, int blocks, int splits, int* status, W4Out o) {
    using S = TcShape<BN, BYTES, G>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::RINGS);     // weights' places full, empty, tokens' full, empty, sums full, empty
    constexpr int FULL = 0, EMPTY = S::STAGES, ROWS_FULL = 2 * S::STAGES, ROWS_EMPTY = ROWS_FULL + S::ROWS, SUM_FULL = ROWS_EMPTY + S::ROWS;
    constexpr int SUM_EMPTY = SUM_FULL + S::BUFS, BARS = SUM_EMPTY + S::BUFS;
    static_assert(BARS * 8 + 4 <= 512, "room for the barriers");
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + BARS);
    float* scales = reinterpret_cast<float*>(smem + S::RINGS + 512);     // 8-bit rows: [group][token]
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
        for (int i = 0; i < 2 * S::ROWS; ++i) mbar_init(smem_u32(&bars[ROWS_FULL + i]), 1);
        for (int i = 0; i < S::BUFS; ++i) {
            mbar_init(smem_u32(&bars[SUM_FULL + i]), 1);
            mbar_init(smem_u32(&bars[SUM_EMPTY + i]), 8);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
    }
    if (warp == 1) {
        tcgen05_alloc(smem_u32(tmem_slot), S::TMEM);
        tcgen05_relinquish();
    }
    // the widening warps' weights: stages phase, phase + WIDENS, ... of a tile of 16 rows, AHEAD of them in registers before anything is waited for
    const int wide = warp - 2, tile = min(row0 / 16 + (wide & 7), tiles - 1), phase = wide >> 3;        // (rows that are not there: some others)
    const bool widens = wide >= 0 && wide < 8 * S::WIDENS;
    constexpr int STEP = S::WIDENS * S::BLOCKS;          // blocks from one of a warp's stages to its next
    const int block0 = (from + phase) * S::BLOCKS, stages = widens ? (n - phase + S::WIDENS - 1) / S::WIDENS : 0;
    const uint4* next_w = w0 + ((size_t)tile * blocks + block0) * 32 + lane;
    const uint32_t* next_s = w1 + ((size_t)tile * all_groups + block0 * 64 / G) * 8 + (lane >> 2);
    uint4 w[S::AHEAD][S::BLOCKS];
    uint32_t sc[S::AHEAD][S::SCALES ? S::SCALES : 1];
    int asked = 0;
    auto ask = [&](int into) {
        if (asked < stages) {
            w[into][0] = *next_w;
            if constexpr (S::BLOCKS == 2)                // (the last stage's second block may not be there)
                w[into][1] = asked + 1 < stages || block0 + S::BLOCKS * stages <= blocks ? next_w[32] : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
            for (int p = 0; p < S::SCALES; ++p) sc[into][p] = next_s[8 * p];
            next_w += 32 * STEP;
            if constexpr (S::SCALES > 0) next_s += 8 * STEP * 64 / G;                   // (two stages on are whole groups on)
            ++asked;
        }
    };
#pragma unroll
    for (int i = 0; i < S::AHEAD; ++i) ask(i);
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem = *tmem_slot;

    const int add = warp - 10, quarter = warp & 3, cols0 = add >= 4 ? BN / 2 : 0;       // adding warps: 32 rows, half the tokens
    Two acc[BYTES ? BN / 4 : 1] = {};
    bool ok = true;
    if (warp == 0) {
        // ---------------- the tokens' numbers
        if (lane == 0) {
            pdl_wait();
            const uint32_t full = smem_u32(&bars[ROWS_FULL]), empty = smem_u32(&bars[ROWS_EMPTY]), to = smem_u32(smem) + S::STAGES * S::A;
            for (int i = 0; i < n; i += 8) {
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    if (i + u >= n || !ok) break;
                    const int at = u % S::ROWS;
                    if (i > 0 || u >= S::ROWS) ok = wait_for(empty + 8 * at, (S::ROWS == 8 ? i / 8 & 1 : u / S::ROWS & 1) ^ 1, &abort_flag);
                    if (!ok) break;
                    mbar_expect_tx(full + 8 * at, S::B);
                    tma_load_2d(to + at * S::B, &map_x, (from + i + u) * S::BLOCKS * 64, tok0, full + 8 * at);
                }
            }
        }
    } else if (warp == 1) {
        // ---------------- the products
        // Eight stages a turn, after which every ring is back where it was: places, parities and descriptors are constants.  (With remainders and
        // addresses formed anew this one thread, not the tensor cores, was the limit: 400 cycles a stage, whatever the tile.)
        if (elect_one()) {
            const uint32_t full = smem_u32(&bars[FULL]), empty = smem_u32(&bars[EMPTY]), rows_full = smem_u32(&bars[ROWS_FULL]), rows_empty = smem_u32(&bars[ROWS_EMPTY]);
            const uint32_t sum_full = smem_u32(&bars[SUM_FULL]), sum_empty = smem_u32(&bars[SUM_EMPTY]);
            const uint64_t da0 = make_smem_desc(smem_u32(smem)), db0 = make_smem_desc(smem_u32(smem) + S::STAGES * S::A);
            for (int i = 0; i < n && ok; i += 8) {
                const uint32_t turn = i / 8 & 1;
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    if (i + u >= n) break;
                    const int a = u % S::STAGES, r = u % S::ROWS;
                    ok = wait_for(rows_full + 8 * r, S::ROWS == 8 ? turn : u / S::ROWS & 1, &abort_flag) && wait_for(full + 8 * a, u / S::STAGES & 1, &abort_flag);
                    if (!ok) break;
                    tcgen05_fence_after();
                    const uint64_t da = da0 + a * (S::A / 16), db = db0 + r * (S::B / 16);
                    if constexpr (BYTES) {
#pragma unroll
                        for (int p = 0; p < S::PARTS; ++p) {
                            const int sum = u * S::PARTS + p, buf = sum % S::BUFS;
                            if (i > 0 || sum >= S::BUFS) {
                                ok = wait_for(sum_empty + 8 * buf, (sum / S::BUFS & 1) ^ 1, &abort_flag);
                                if (!ok) break;
                                tcgen05_fence_after();
                            }
#pragma unroll
                            for (int k = 0; k < 4 / S::PARTS; ++k) {                    // 32 columns an instruction
                                const int at = 2 * (p * (4 / S::PARTS) + k);
                                mma_step<BN, BYTES>(tmem + buf * BN, da + at, db + at, k ? 1u : 0u);
                            }
                            tcgen05_commit(sum_full + 8 * buf);
                        }
                        if (!ok) break;
                    } else {
#pragma unroll
                        for (int k = 0; k < 4; ++k) mma_step<BN, BYTES>(tmem, da + 2 * k, db + 2 * k, (i | u | k) ? 1u : 0u);        // 16 columns
                    }
                    tcgen05_commit(empty + 8 * a);
                    tcgen05_commit(rows_empty + 8 * r);
                }
            }
            if (!BYTES) tcgen05_commit(sum_full);
        }
    } else if (widens) {
        // ---------------- the weights
        const int g = lane >> 2, t = lane & 3;
        const bool odd = g & 1;
        const uint32_t row = smem_u32(smem) + (16 * (wide & 7) + g) * 128;              // (rows of 128 bytes, 16-byte pieces swapped by row % 8 = g)
        const uint32_t full = smem_u32(&bars[FULL + phase]), empty = smem_u32(&bars[EMPTY + phase]);
        // where this lane's pieces of a stage go: by the row's parity the other half (8-bit rows: block) first, and rows' pieces meet all banks
        uint32_t place[BYTES ? 4 : 2];
        if constexpr (BYTES) {
#pragma unroll
            for (int j = 0; j < 4; ++j) place[j] = row + (((4 * (odd ^ (j >> 1)) + 2 * (j & 1) + (t >> 1)) ^ g) * 16) + (t & 1) * 8;
        } else {
#pragma unroll
            for (int j = 0; j < 2; ++j) place[j] = row + (((4 * (odd ^ j) + t) ^ g) * 16);
        }
        uint32_t parity = 1;
        for (int done = 0; done < stages && ok;) {
#pragma unroll
            for (int u = 0; u < S::AHEAD; ++u, ++done) {
                if (done >= stages) break;
                const uint32_t to = phase * S::A + u % S::TURN * S::WIDENS * S::A;
                if (done >= S::TURN) {
                    ok = wait_for(empty + u % S::TURN * S::WIDENS * 8, parity, &abort_flag);
                    if (!ok) break;
                }
                if constexpr (BYTES) {
                    const uint4 v[2] = {odd ? w[u][1] : w[u][0], odd ? w[u][0] : w[u][1]};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t m = 0xf0f0f0f0u, lo = j & 1 ? v[j >> 1].y : v[j >> 1].x, hi = j & 1 ? v[j >> 1].w : v[j >> 1].z;
                        to_shared8(place[j] + to, lo << 4 & m, lo & m);
                        to_shared8(place[j] + to + 1024, hi << 4 & m, hi & m);
                    }
                } else {
                    const uint4 v = w[u][0];
                    const uint32_t lo[2] = {odd ? v.y : v.x, odd ? v.x : v.y}, hi[2] = {odd ? v.w : v.z, odd ? v.z : v.w};
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const uint32_t s2 = S::SCALES == 2 ? (odd ^ j ? sc[u][S::SCALES - 1] : sc[u][0]) : sc[u][0];
                        four_pairs(place[j] + to, lo[j], __byte_perm(s2, 0, 0x1010));
                        four_pairs(place[j] + to + 1024, hi[j], __byte_perm(s2, 0, 0x3232));
                    }
                }
                ask(u);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) at_arrive(full + u % S::TURN * S::WIDENS * 8);
                if (u % S::TURN == S::TURN - 1) parity ^= 1;
            }
        }
    }
    pdl_wait(xs);                                        // (whoever writes from here on has waited)
    if (add >= 0) {
        // ---------------- the sums
        const int row = row0 + 32 * quarter + lane;
        if constexpr (BYTES) {
            const int first = from * S::PARTS, count = n * S::PARTS;
            for (int i = threadIdx.x - 320; i < count * live; i += 256) {
                const int tok = i / count, gr = i - tok * count;
                scales[gr * BN + tok] = first + gr < all_groups ? xs[(size_t)(tok0 + tok) * all_groups + first + gr] : 0.f;
            }
            asm volatile("bar.sync 1, 256;" ::: "memory");
            // this row's scales; what lies behind the last row or group is read from it and meets tokens' scales of zero, or is not written
            const int r = min(row, 16 * tiles - 1);
            const __nv_bfloat16* ws = reinterpret_cast<const __nv_bfloat16*>(w1) + ((size_t)(r / 16) * all_groups + first) * 16 + 2 * (r % 8) + r % 16 / 8;
            const int last = all_groups - 1 - first;
            float next[S::BUFS];
#pragma unroll
            for (int u = 0; u < S::BUFS; ++u) next[u] = __bfloat162float(ws[(size_t)min(u, last) * 16]);
            const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16) + cols0, sum_full = smem_u32(&bars[SUM_FULL]), sum_empty = smem_u32(&bars[SUM_EMPTY]);
            const float* a = scales + cols0;
            uint32_t parity = 0;
            for (int i = 0; i < count && ok; i += S::BUFS, parity ^= 1) {
#pragma unroll
                for (int u = 0; u < S::BUFS; ++u, a += BN) {
                    if (i + u >= count) break;
                    const float f = next[u] * 0.0625f;   // (the products hold 16 q)
                    const Two ff = two(f, f);
                    next[u] = __bfloat162float(ws[(size_t)min(i + u + S::BUFS, last) * 16]);
                    ok = wait_for(sum_full + 8 * u, parity, &abort_flag);
                    if (!ok) break;
                    tcgen05_fence_after();
                    constexpr int CH = BN == 64 ? 32 : 16;              // (32 numbers beside 64 sums would not fit the registers)
#pragma unroll
                    for (int c = 0; c < BN / 2; c += CH) {
                        uint32_t r[CH];
                        if constexpr (CH == 32) tcgen05_ld32(lanes + u * BN + c, r);
                        else tcgen05_ld16(lanes + u * BN + c, r);
                        tcgen05_wait_ld();
                        if (c + CH == BN / 2) {
                            tcgen05_fence_before();
                            __syncwarp();
                            if (lane == 0) at_arrive(sum_empty + 8 * u);
                        }
#pragma unroll
                        for (int j = 0; j < CH; j += 4) {
                            const float4 x = *reinterpret_cast<const float4*>(a + c + j);
                            const Two v0 = two((float)(int)r[j], (float)(int)r[j + 1]), v1 = two((float)(int)r[j + 2], (float)(int)r[j + 3]);        // (exact)
                            acc[(c + j) / 2] = fma2(v0, mul2(two(x.x, x.y), ff), acc[(c + j) / 2]);
                            acc[(c + j) / 2 + 1] = fma2(v1, mul2(two(x.z, x.w), ff), acc[(c + j) / 2 + 1]);
                        }
                    }
                }
            }
        } else if (n > 0) {
            ok = wait_for(smem_u32(&bars[SUM_FULL]), 0, &abort_flag);
            tcgen05_fence_after();
        }
    }
    __syncwarp();
    // a cluster's sums go through the stages' place; one CTA's straight out
    if (splits > 1) __syncthreads();                     // (the last sums were there: every product has read its stages)
    if (add >= 0 && ok) {
        float* sums = reinterpret_cast<float*>(smem) + 32 * quarter + lane;
        const int row = row0 + 32 * quarter + lane;
        auto give = [&](int tok, float v) {
            if (splits > 1) sums[tok * W4T_PITCH] = v;
            else if (tok < live) w4_write(o, tok0 + tok, row, v);
        };
        if constexpr (BYTES) {
#pragma unroll
            for (int j = 0; j < BN / 4; ++j) {
                float a, b;
                one(acc[j], a, b);
                give(cols0 + 2 * j, a);
                give(cols0 + 2 * j + 1, b);
            }
        } else {
            constexpr int CH = BN / 2 < 32 ? 16 : 32;
#pragma unroll 1
            for (int c = 0; c < BN / 2; c += CH) {
                uint32_t r[CH];
                const uint32_t at = tmem + ((uint32_t)(quarter * 32) << 16) + cols0 + c;
                if (n > 0) {
                    if constexpr (CH == 32) tcgen05_ld32(at, r); else tcgen05_ld16(at, r);
                    tcgen05_wait_ld();
                }
#pragma unroll
                for (int j = 0; j < CH; ++j) give(cols0 + c + j, n > 0 ? __uint_as_float(r[j]) : 0.f);
            }
        }
    }
    if (splits > 1) {
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        const float* sums = reinterpret_cast<const float*>(smem);
        for (int i = rank * W4T_THREADS + threadIdx.x; i < live * 128; i += splits * W4T_THREADS) {
            const int tok = i / 128, r = i % 128;
            const uint32_t here = smem_u32(sums + tok * W4T_PITCH + r);
            float v = 0.f;
            for (int c = 0; c < splits; ++c) {
                uint32_t there;
                float f;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(here), "r"(c));
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(f) : "r"(there) : "memory");
                v += f;
            }
            if (!abort_flag) w4_write(o, tok0 + tok, row0 + r, v);
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

// ---------------------------------------------------------------- host side
// [rows, cols] of 1- or 2-byte numbers, ld apart; a box is 128 bytes of box_rows rows, pieces of 16 bytes swapped as the MMA wants them.
static int rows_map(CUtensorMap* map, const void* base, long long rows, long long cols, long long ld, int bytes, int box_rows) {
    EncodeTiledFn f = encode_fn();
    if (!f) return RF_ERR_UNSUPPORTED;
    if ((reinterpret_cast<uintptr_t>(base) & 15) || (ld * bytes) % 16) return RF_ERR_BAD_ARG;
    cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)(ld * bytes)};
    cuuint32_t box[2] = {(cuuint32_t)(128 / bytes), (cuuint32_t)box_rows}, steps[2] = {1, 1};
    const CUresult r = f(map, bytes == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box, steps,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : RF_ERR_BAD_ARG;
}

template <int BN, bool BYTES, int G>
static int tc_shared(int blocks, int splits) {
    using S = TcShape<BN, BYTES, G>;
    const int all = (blocks + S::BLOCKS - 1) / S::BLOCKS, most = (all + splits - 1) / splits;
    return S::FIXED + (BYTES ? most * S::PARTS * BN * 4 : 0);
}
// f(tokens of a tile, 8-bit rows, group) as constants; false where there is no such kernel
template <typename F>
static bool with_tc(int bn, int x_kind, int G, F f) {
    auto by_group = [&](auto b, auto bytes) {
        if (G == 32) f(b, bytes, std::integral_constant<int, 32>());
        else if (G == 64) f(b, bytes, std::integral_constant<int, 64>());
        else f(b, bytes, std::integral_constant<int, 128>());
    };
    auto by_kind = [&](auto b) {
        if (x_kind == 0) by_group(b, std::true_type());
        else by_group(b, std::false_type());
    };
    if (bn == 32) by_kind(std::integral_constant<int, 32>());
    else if (bn == 64) by_kind(std::integral_constant<int, 64>());
    else if (bn == 128) by_kind(std::integral_constant<int, 128>());
    else return false;
    return true;
}
#define W4T_MOST_SHARED (226 * 1024)                  // (the abort flag has a place of its own)

extern "C" {

// Bytes of shared memory that a block takes with tiles of bn tokens and a share of the columns in `splits` (0: no such kernel).
int rf_gemm_w4_tc_shared(int x_kind, int K, int G, int bn, int splits) {
    if (K <= 0 || bad_group(G) || splits < 1) return 0;
    int bytes = 0;
    const int blocks = padded(K, G) / 64;
    with_tc(bn, x_kind, G, [&](auto b, auto kind, auto g) { bytes = tc_shared<decltype(b)::value, decltype(kind)::value, decltype(g)::value>(blocks, splits); });
    return bytes;
}

// As rf_gemm_w4 (quantized.cu), with tiles of bn tokens (32, 64, 128); 16-bit rows must start on 16 bytes and lie whole 16 bytes apart.
int rf_gemm_w4_tc(int x_kind, const void* x, const void* xs, long long ldx, const void* packed, const void* scales, const void* bias, int bias_is_f32,
                  void* out, int out_is_f32, int add, int bn, int splits, int M, int N, int K, int G, int* status, cudaStream_t st) {
    if (M <= 0 || N <= 0 || K <= 0 || bad_group(G) || (add && !out_is_f32) || splits < 1 || splits > 8) return RF_ERR_BAD_ARG;
    if (!aligned(packed, 16) || !aligned(scales, 16)) return RF_ERR_BAD_ARG;
    const int Kp = padded(K, G), blocks = Kp / 64;
    const long long x_blocks = (long long)((N + 127) / 128) * splits, y = (M + (long long)bn - 1) / (bn > 0 ? bn : 1);
    if (x_blocks > 0x7fffffffll || y > 65535) return RF_ERR_UNSUPPORTED;
    CUtensorMap map;
    if (const int e = rows_map(&map, x, M, x_kind == 0 ? Kp : K, ldx, x_kind == 0 ? 1 : 2, bn)) return e;
    const W4Out o{out, bias, bias_is_f32, out_is_f32, add, M, N};
    int bad = 0;
    const bool known = with_tc(bn, x_kind, G, [&](auto b, auto kind, auto g) {
        constexpr int BN = decltype(b)::value, GC = decltype(g)::value;
        constexpr bool BYTES = decltype(kind)::value;
        const int smem = tc_shared<BN, BYTES, GC>(blocks, splits);
        if (smem > W4T_MOST_SHARED) { bad = RF_ERR_UNSUPPORTED; return; }
        static PerDevice<bool> set;
        bool& done = set.here();
        if (!done) {
            const cudaError_t e = cudaFuncSetAttribute(w4_tc_kernel<BN, BYTES, GC>, cudaFuncAttributeMaxDynamicSharedMemorySize, W4T_MOST_SHARED);
            if (e != cudaSuccess) { bad = (int)e; return; }
            done = true;
        }
        const dim3 grid((unsigned)x_blocks, (unsigned)y), block(W4T_THREADS);
        auto go = [&](auto... args) {
            if (splits > 1) rf_launch_cluster(w4_tc_kernel<BN, BYTES, GC>, grid, block, smem, st, splits, args...);
            else rf_launch(w4_tc_kernel<BN, BYTES, GC>, grid, block, smem, st, args...);
        };
        go(map, (const uint4*)packed, (const uint32_t*)scales, (const float*)xs, blocks, splits, status, o);
    });
    if (!known) return RF_ERR_BAD_ARG;
    if (bad) return bad;
    RF_LAUNCH_CHECK();
    return 0;
}

}  // extern "C"
