// Products of bfloat16 rows with 4-bit weights on the 5th-generation tensor cores, from some 17 tokens on.
//
// Weights are the accumulator's rows, tokens its columns.  128 rows' weights come as they are stored, by TMA, four blocks of 128 columns a stage,
// ahead and before the wait for the kernel before.  Four groups of four warps have every fourth block each: a lane reads a row's (whatever the
// order in which the result's rows then lie), widens them to bfloat16 numbers, scale and all (exactly, with scales of five significant bits;
// others are rounded), and writes them into tensor memory, where the MMA takes its first operand from.  (Through shared memory instead,
// writing them there and the MMA's reading them were the limit: 64 x 37,888 x 3,584 33.7 us.)  The tokens' numbers come by TMA into a ring of
// their own.  Long rows are shared out to the CTAs of a cluster, which add up their sums through shared memory in the order of their ranks.
//
// The tensor cores cut what an addition loses instead of rounding it, and what is cut adds up (1,999 x 3,584 x 18,944 against 64 bits: one sum
// 1.1e-5 off, pieces of 6,315 columns 2.6e-6).  For 32-bit results a sum runs over W4T_PIECE columns at most: the widening warps add it to a
// second one beside it, rounded, while the next piece goes into another accumulator (tiles of 128 tokens: into the same one, after a wait).
//
// What it took (32-bit results, device time in a chain of launches over weights larger than L2): 32 x 37,888 x 3,584 28.5 us, 64 30.2, 128 38.5 (the
// 16-bit product of as many tokens 42, 44, 49), 64 x 3,584 x 18,944 20.2 (81), 128 x 4,608 x 3,584 11.7 (22.4), 512 x 3,584 x 18,944 68 (94).
// What bounds it: up to 128 tokens the widening, 1.5 us for 512 columns of 128 rows (15 instructions a lane for 8 weights; the schedulers issue in
// 56 to 60 % of cycles, waits between its parts), and what comes before and after a block's loop, 3 us and, with 128 tokens, 7; many tokens: widening
// beside MMAs that would take 1.1 us.
//
// Every wait on an mbarrier is bounded (2 s): status word 13.
#include <type_traits>
#include "quantized.cuh"
#include "tcgen05_common.cuh"

#define W4T_THREADS (32 * 20)                            // the tokens' producer, the MMA issuer, the weights' producer, one idle, sixteen widening warps
#define W4T_PIECE 2048                                   // columns of one sum where the result is 32-bit
#define W4T_PITCH (128 + 4)                              // of the sums that a cluster exchanges, [token][row]
#define W4T_MOST_SHARED (226 * 1024)                     // (the abort flag has a place of its own)

template <int BN, int G>
struct TcShape {
    static constexpr int GROUPS = 4, STORED = 8;         // of widening warps; a stage's blocks of 64 columns as they are stored
    static constexpr int WORDS = STORED * 512, SCALES = 512 / G * 32, STAGES = 2;       // bytes of a stage, of a tile of 16 rows
    static constexpr int PLACES = 4, ROWS = BN == 128 ? 4 : 8;          // blocks of 128 columns in tensor memory; of tokens' numbers
    static constexpr int B = BN * 256, RINGS = ROWS * B + STAGES * 8 * (WORDS + SCALES), NEEDED = 1024 + RINGS + 512;     // (alignment, barriers)
    static constexpr int BUFS = BN == 128 ? 1 : 2, SUMS = 64 * PLACES;  // accumulators and, behind them, the pieces' sum, behind the weights
    static constexpr int SHARE = BN / 4 < 16 ? 16 : BN / 4;             // a widening warp's part of the sums: 32 rows, so many tokens
    static constexpr int PIECE = W4T_PIECE / 128, PIECE_STAGES = PIECE / GROUPS;
    // A block takes all of an SM's tensor memory.  It asks for so much shared memory that no block of another kernel that wants some fits beside it:
    // two clusters could otherwise wait for one another's.
    static constexpr int BYTES = NEEDED > 190 * 1024 ? NEEDED : 190 * 1024;
    static_assert(BYTES <= W4T_MOST_SHARED && RINGS >= BN * W4T_PITCH * 4, "the rings' place holds the sums");
    static_assert(SUMS + (BUFS + 1) * BN <= 512 && PIECE % ROWS == 0, "");
    static_assert(PLACES % GROUPS == 0 && ROWS % GROUPS == 0, "one parity bit tells two phases apart, not three");
};

// Bounded wait as mbar_wait, asleep between looks: what waits here waits long, and the widening warps need the issue slots.  (The clock is
// not read before the first sleep has ended without what it was for.)
__device__ __forceinline__ bool look_asleep(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(bar), "r"(parity), "r"(20000u) : "memory");
    return ok;
}
__device__ __noinline__ bool wait_asleep(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
    const unsigned long long t0 = global_ns();
    while (!look_asleep(bar, parity)) {
        if (*abort_flag) return false;
        if (global_ns() - t0 > TC_WAIT_LIMIT_NS) { *abort_flag = 1; return false; }
    }
    return true;
}
__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
    return look_asleep(bar, parity) || wait_asleep(bar, parity, abort_flag);
}
// After a wait that gave up: until the last `places` of `asked` copies have landed (a limited wait), so that none comes after the block's end.
__device__ __noinline__ void let_land(uint32_t full, int places, int asked) {
    int never = 0;
    for (int i = asked > places ? asked - places : 0; i < asked; ++i) wait_asleep(full + 8 * (i % places), i / places & 1, &never);
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(bar) : "memory");
}
// An arrival of the lanes with `mine` (a predicate, no branch: the warp stays together for the reads and writes of tensor memory behind it).
__device__ __forceinline__ void at_arrive_if(uint32_t bar, bool mine) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "@p mbarrier.arrive.shared::cta.b64 _, [%0];\n\t}"
        ::"r"(bar), "r"((uint32_t)mine) : "memory");
}
__device__ __forceinline__ uint2 shared8(uint32_t at) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at));
    return v;
}
__device__ __forceinline__ uint32_t shared2(uint32_t at) {
    uint16_t v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at));
    return v;
}

// Eight columns, a word's, as bfloat16 numbers times a scale: bytes q + 8 below 0x43 are 128 + q + 8, less 136.
__device__ __forceinline__ void widen(uint32_t* out, uint32_t w, __nv_bfloat162 s) {
    const uint32_t low = (w & 0x0f0f0f0fu) ^ 0x08080808u, high = (w >> 4 & 0x0f0f0f0fu) ^ 0x08080808u;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        uint32_t v = __byte_perm(j & 2 ? high : low, 0x43434343u, j & 1 ? 0x4342 : 0x4140);
        const __nv_bfloat162 r = __hmul2(__hadd2(*reinterpret_cast<__nv_bfloat162*>(&v), __float2bfloat162_rn(-136.f)), s);
        out[j] = *reinterpret_cast<const uint32_t*>(&r);
    }
}

// The row of the block that a lane of a warp has (accumulators' rows 32 (warp & 3) + lane).
__device__ __forceinline__ int row_of(int warp, int lane) { return 32 * (warp & 3) + 8 * (lane & 3) + (lane >> 2); }

// A widening warp's share of a piece's sum added to the sum of those before.
template <int BN, int G>
__device__ __noinline__ bool add_piece(uint32_t tmem, uint32_t sum_full, int piece, volatile int* abort_flag) {
    using S = TcShape<BN, G>;
    const int buf = piece % S::BUFS, warp = threadIdx.x >> 5, share = (warp - 4) / 4 * S::SHARE;
    if (!__all_sync(0xffffffffu, wait_for(sum_full + 8 * buf, piece / S::BUFS & 1, abort_flag))) return false;
    tcgen05_fence_after();
    if (share < BN) {
        const uint32_t rows = tmem + ((uint32_t)((warp & 3) * 32) << 16) + S::SUMS + share;
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
    at_arrive_if(sum_full + 8 * (S::BUFS + buf), (threadIdx.x & 31) == 0);
    return true;
}

// A lane's row of sixteen tokens (from c on) of the result: the last piece's sum and that of those before, into `sums` ([token][row]) or, without,
// straight out.  (Functions of their own keep these parts' registers out of the loop over the weights.)
__device__ __noinline__ void write_16(uint32_t last_sum, uint32_t sum_before, bool any, bool more, float* sums, int row0, int c, int tok0, int live, W4Out o) {
    uint32_t r[16], before[16];
    if (any) tcgen05_ld16(last_sum + c, r);
    if (more) tcgen05_ld16(sum_before + c, before);
    const int at_row = row_of(threadIdx.x >> 5, threadIdx.x & 31), row = row0 + at_row;
    const bool there = row < o.N;
    const size_t to = (size_t)(tok0 + c) * o.N + row;
    const float bias = there && o.bias != nullptr ? load_vec(o.bias, o.bias_is_f32, row) : 0.f;
    float old[16];
    if (sums == nullptr && o.add) {                      // (all at once: a load after every store would wait for it)
#pragma unroll
        for (int j = 0; j < 16; ++j) old[j] = there && c + j < live ? reinterpret_cast<const float*>(o.out)[to + (size_t)j * o.N] : 0.f;
    }
    __syncwarp();                                        // (rows that are not there have read nothing)
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
    __syncwarp();                                        // (... nor written anything: the next sixteen tokens' reads need the whole warp)
}

template <int BN, int G>
__global__ void __launch_bounds__(W4T_THREADS, 1) w4_tc_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                                                               const __grid_constant__ CUtensorMap map_s, int blocks, int splits, bool pieces, int* status, W4Out o) {
    using S = TcShape<BN, G>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t rows_at = smem_u32(smem), weights_at = rows_at + S::ROWS * S::B, scales_at = weights_at + S::STAGES * 8 * S::WORDS, bars = rows_at + S::RINGS;
    // stages of weights full, empty; blocks in tensor memory full, tokens' numbers full, a block's products done; sums full, read; every product done
    constexpr int W_FULL = 0, W_EMPTY = W_FULL + 8 * S::STAGES, A_FULL = W_EMPTY + 8 * S::STAGES, X_FULL = A_FULL + 8 * S::PLACES;
    constexpr int DONE = X_FULL + 8 * S::ROWS, S_FULL = DONE + 8 * S::ROWS, S_READ = S_FULL + 8 * S::BUFS, END = S_READ + 8 * S::BUFS;
    static_assert(END + 8 <= 512, "room for the barriers");
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;
    pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = blockIdx.x % splits, row0 = blockIdx.x / splits * 128, tok0 = blockIdx.y * BN, live = min(BN, o.M - tok0);
    // stages of four blocks, the last one of a row with what is left
    const int all = (blocks + S::STORED - 1) / S::STORED, from = (int)((long long)all * rank / splits), n = (int)((long long)all * (rank + 1) / splits) - from;
    const int nb = n > 0 ? (min(S::STORED * n, blocks - S::STORED * from) + 1) / 2 : 0;
    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int i = 0; i < S::PLACES; ++i) mbar_init(bars + A_FULL + 8 * i, 4);
        for (int i = 0; i < S::ROWS; ++i) mbar_init(bars + X_FULL + 8 * i, 1), mbar_init(bars + DONE + 8 * i, 1);
        for (int i = 0; i < S::BUFS; ++i) mbar_init(bars + S_FULL + 8 * i, 1), mbar_init(bars + S_READ + 8 * i, 16);
        mbar_init(bars + END, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
    }
    auto ask_weights = [&](int i) {
        const int at = i % S::STAGES;
        mbar_expect_tx(bars + W_FULL + 8 * at, 8 * (S::WORDS + S::SCALES));
        tma_load_3d(weights_at + at * 8 * S::WORDS, &map_w, 0, (from + i) * S::STORED * 4, row0 / 16, bars + W_FULL + 8 * at);
        tma_load_2d(scales_at + at * 8 * S::SCALES, &map_s, (from + i) * (S::SCALES / 2), row0 / 16, bars + W_FULL + 8 * at);
    };
    if (warp == 2 && lane == 0) {                        // (the first before anything else)
        for (int i = 0; i < S::STAGES; ++i) mbar_init(bars + W_FULL + 8 * i, 1), mbar_init(bars + W_EMPTY + 8 * i, 16);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        for (int i = 0; i < min(n, S::STAGES); ++i) ask_weights(i);
    }
    if (warp == 3) {
        tcgen05_alloc(smem_u32(&tmem_slot), 512);
        tcgen05_relinquish();
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem = tmem_slot;
    const int last = pieces && nb > 0 ? (nb - 1) / S::PIECE : 0;         // the piece that the result is read from, with the sum of those before
    bool ok = true;
    if (warp == 0) {
        // ---------------- the tokens' numbers
        if (lane == 0) {
            pdl_wait();
            int i = 0;
            for (; i < nb; ++i) {
                const int at = i % S::ROWS, column = (from * S::GROUPS + i) * 128;
                if (i >= S::ROWS && !wait_for(bars + DONE + 8 * at, (i / S::ROWS & 1) ^ 1, &abort_flag)) break;
                mbar_expect_tx(bars + X_FULL + 8 * at, S::B);
                tma_load_2d(rows_at + at * S::B, &map_x, column, tok0, bars + X_FULL + 8 * at);
                tma_load_2d(rows_at + at * S::B + S::B / 2, &map_x, column + 64, tok0, bars + X_FULL + 8 * at);
            }
            if (i < nb) let_land(bars + X_FULL, S::ROWS, i);
        }
    } else if (warp == 2) {
        // ---------------- the weights (sixteen bulk copies a stage, a tile's weights and scales each, took 1,800 cycles to issue)
        if (lane == 0) {
            int i = min(n, S::STAGES);
            for (; i < n; ++i) {
                if (!wait_for(bars + W_EMPTY + 8 * (i % S::STAGES), (i / S::STAGES & 1) ^ 1, &abort_flag)) break;
                ask_weights(i);
            }
            if (i < n) let_land(bars + W_FULL, S::STAGES, i);
        }
    } else if (warp == 1) {
        // ---------------- the products
        // ROWS blocks a turn, after which every ring is back where it was: places and descriptors are constants.
        if (elect_one()) {
            const uint64_t db0 = make_smem_desc(rows_at);
            uint32_t sum = tmem + S::SUMS;
            bool starts = true;
            for (int i = 0; i < nb && ok; i += S::ROWS, starts = false) {
                if (pieces && i > 0 && i % S::PIECE == 0) {
                    const int piece = i / S::PIECE, buf = piece % S::BUFS;
                    tcgen05_commit(bars + S_FULL + 8 * ((piece - 1) % S::BUFS));
                    if (piece >= S::BUFS) ok = wait_for(bars + S_READ + 8 * buf, piece / S::BUFS - 1 & 1, &abort_flag);
                    if (!ok) break;
                    tcgen05_fence_after();
                    sum = tmem + S::SUMS + buf * BN;
                    starts = true;
                }
                const uint32_t turn = i / S::ROWS & 1;
#pragma unroll
                for (int u = 0; u < S::ROWS; ++u) {
                    if (i + u >= nb) break;
                    const int a = u % S::PLACES;
                    ok = wait_for(bars + X_FULL + 8 * u, turn, &abort_flag) && wait_for(bars + A_FULL + 8 * a, S::ROWS == S::PLACES ? turn : u / S::PLACES & 1, &abort_flag);
                    if (!ok) break;
                    tcgen05_fence_after();
#pragma unroll
                    for (int k = 0; k < 8; ++k)          // 16 columns
                        tcgen05_mma_bf16_ts(sum, tmem + a * 64 + k * 8, db0 + (u * S::B + k / 4 * (S::B / 2)) / 16 + 2 * (k % 4), make_idesc(BN), u || k || !starts ? 1u : 0u);
                    tcgen05_commit(bars + DONE + 8 * u);
                }
            }
            tcgen05_commit(bars + END);
            if (!ok) let_land(bars + END, 1, 1);
        }
    } else if (warp >= 4) {
        // ---------------- the weights into tensor memory: a group of warps has every fourth block, a warp 32 rows, a lane one
        const int group = (warp - 4) / 4, g = lane >> 2, t = lane & 3, tile = 2 * (warp & 3) + (t >> 1);
        const uint32_t to = tmem + ((uint32_t)((warp & 3) * 32) << 16) + group * 64;
        // entry 4 g + p of a stored block: rows of 128 bytes, two g each, their pieces of 16 swapped by row % 8
        const uint32_t words_at = weights_at + tile * S::WORDS + group * 1024 + g / 2 * 128 + 8 * (t & 1), piece0 = ((g & 1) * 4 ^ g / 2) * 16;
        const uint32_t scale_at = scales_at + tile * S::SCALES + group * 128 / G * 32 + 4 * g + 2 * (t & 1);
        int summed = 0;
        for (int i = 0; i < n && ok; ++i) {
            if ((i - 1) / S::PIECE_STAGES > summed && summed < last) {  // (a piece is added once the next one's first stage is on its way)
                ok = add_piece<BN, G>(tmem, bars + S_FULL, summed, &abort_flag);
                if (!ok) break;
                ++summed;
            }
            const int at = i % S::STAGES, number = i * S::GROUPS + group;
            ok = __all_sync(0xffffffffu, wait_for(bars + W_FULL + 8 * at, i / S::STAGES & 1, &abort_flag));
            if (!ok || number >= nb) break;
            const uint32_t here = words_at + at * 8 * S::WORDS;
#pragma unroll
            for (int h = 0; h < 2; ++h) {                // stored blocks (rows and columns that are not there: zeros)
                uint32_t out[32];
                const uint32_t its = scale_at + at * 8 * S::SCALES + 64 * h / G * 32;
                uint32_t s0 = shared2(its), s1 = G == 32 ? shared2(its + 32) : s0;
                s0 |= s0 << 16;
                s1 |= s1 << 16;
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                    const uint2 v = shared8(here + 512 * h + (piece0 ^ 64 * h ^ 16 * p));
                    widen(out + 4 * p, v.x, *reinterpret_cast<const __nv_bfloat162*>(&s0));
                    widen(out + 16 + 4 * p, v.y, *reinterpret_cast<const __nv_bfloat162*>(&s1));
                }
                if (h == 1) {
                    __syncwarp();                        // all have read the stage
                    at_arrive_if(bars + W_EMPTY + 8 * at, lane == 0);
                } else if (i > 0) {
                    const int before = number - S::PLACES;
                    ok = __all_sync(0xffffffffu, wait_for(bars + DONE + before % S::ROWS * 8, before / S::ROWS & 1, &abort_flag));
                    if (!ok) break;
                    tcgen05_fence_after();
                }
                tcgen05_st32(to + 32 * h, out);
            }
            if (!ok) break;
            tcgen05_wait_st();
            tcgen05_fence_before();
            __syncwarp();
            at_arrive_if(bars + A_FULL + 8 * group, lane == 0);
        }
        for (; ok && summed < last; ++summed) ok = add_piece<BN, G>(tmem, bars + S_FULL, summed, &abort_flag);
    }
    pdl_wait();                                          // (whoever writes from here on has waited)
    // ---------------- the result: a cluster's sums go through the rings' place, one CTA's straight out
    const int share = (warp - 4) / 4 * S::SHARE;
    const bool writes = warp >= 4 && share < BN;
    if (writes && nb > 0) {
        ok = wait_for(bars + END, 0, &abort_flag) && ok;
        tcgen05_fence_after();
    }
    ok = __all_sync(0xffffffffu, ok);
    if (splits > 1) __syncthreads();                     // (every product is done: the rings have been read)
    if (writes && ok) {
        const uint32_t rows = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + S::SUMS;
#pragma unroll 1
        for (int c = share; c < share + S::SHARE; c += 16)
            write_16(rows + last % S::BUFS * BN, rows + S::BUFS * BN, nb > 0, last > 0, splits > 1 ? reinterpret_cast<float*>(smem) : nullptr, row0, c, tok0, live, o);
    }
    if (splits > 1) {
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        for (int i = rank * W4T_THREADS + threadIdx.x; i < live * 32; i += splits * W4T_THREADS) {
            const int tok = i / 32, r = i % 32 * 4;
            const uint32_t here = rows_at + (tok * W4T_PITCH + r) * 4;
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
    if (warp == 3) {
        tcgen05_fence_after();
        tcgen05_dealloc(tmem, 512);
    }
    if (threadIdx.x == 0 && abort_flag && status) atomicExch(status, 13);
}

// ---------------------------------------------------------------- host side
// The stored weights as rows of 128 bytes, [tiles of 16 rows][4 a block][128], pieces of 16 bytes swapped by row % 8; a box is a stage of eight
// tiles.  Their scales as [tiles][groups of 16].
static int weights_map(CUtensorMap* map, const void* base, long long tiles, long long blocks, int stored) {
    EncodeTiledFn f = encode_fn();
    if (!f) return RF_ERR_UNSUPPORTED;
    cuuint64_t dims[3] = {128, (cuuint64_t)(4 * blocks), (cuuint64_t)tiles}, strides[2] = {128, (cuuint64_t)(512 * blocks)};
    cuuint32_t box[3] = {128, (cuuint32_t)(4 * stored), 8}, steps[3] = {1, 1, 1};
    const CUresult r = f(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : RF_ERR_BAD_ARG;
}
static int scales_map(CUtensorMap* map, const void* base, long long tiles, long long groups, int groups_of_stage) {
    EncodeTiledFn f = encode_fn();
    if (!f) return RF_ERR_UNSUPPORTED;
    cuuint64_t dims[2] = {(cuuint64_t)(16 * groups), (cuuint64_t)tiles}, strides[1] = {(cuuint64_t)(32 * groups)};
    cuuint32_t box[2] = {(cuuint32_t)(16 * groups_of_stage), 8}, steps[2] = {1, 1};
    const CUresult r = f(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : RF_ERR_BAD_ARG;
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
    else return false;
    return true;
}

extern "C" {

// out = x w^T (+ bias): x bfloat16 [M, K], rows ldx apart, whole 16 bytes on 16-byte boundaries; out as W4Out has it.  bn: tokens of a tile (32, 64,
// 128); splits: CTAs of a cluster that share out the columns (1 .. 8).
int rf_gemm_w4_tc(const void* x, long long ldx, const void* packed, const void* scales, const void* bias, int bias_is_f32, void* out, int out_is_f32, int add,
                  int bn, int splits, int M, int N, int K, int G, int* status, cudaStream_t st) {
    if (M <= 0 || N <= 0 || K <= 0 || bad_group(G) || (add && !out_is_f32) || splits < 1 || splits > 8 || bn < 1) return RF_ERR_BAD_ARG;
    if (!aligned(packed, 16) || !aligned(scales, 16) || ldx < K) return RF_ERR_BAD_ARG;
    const int blocks = padded(K, G) / 64;
    const long long tiles = ((long long)N + 15) / 16, x_blocks = (tiles + 7) / 8 * splits, y = (M + (long long)bn - 1) / bn;
    if (x_blocks > 0x7fffffffll || y > 65535) return RF_ERR_UNSUPPORTED;
    CUtensorMap map_x, map_w, map_s;
    if (const int e = make_map(&map_x, x, M, K, ldx, bn)) return e;
    const W4Out o = w4_out(out, bias, bias_is_f32, out_is_f32, add, M, N);
    int bad = 0;
    const bool known = with_tc(bn, G, [&](auto b, auto g) {
        constexpr int BN = decltype(b)::value, GC = decltype(g)::value;
        using S = TcShape<BN, GC>;
        if ((bad = weights_map(&map_w, packed, tiles, blocks, S::STORED)) || (bad = scales_map(&map_s, scales, tiles, (long long)blocks * 64 / GC, 64 * S::STORED / GC))) return;
        static PerDevice<bool> set;
        bool& done = set.here();
        if (!done) {
            const cudaError_t e = cudaFuncSetAttribute(w4_tc_kernel<BN, GC>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::BYTES);
            if (e != cudaSuccess) { bad = (int)e; return; }
            done = true;
        }
        const dim3 grid((unsigned)x_blocks, (unsigned)y), block(W4T_THREADS);
        auto go = [&](auto... args) {
            if (splits > 1) rf_launch_cluster(w4_tc_kernel<BN, GC>, grid, block, S::BYTES, st, splits, args...);
            else rf_launch(w4_tc_kernel<BN, GC>, grid, block, S::BYTES, st, args...);
        };
        go(map_x, map_w, map_s, blocks, splits, out_is_f32 != 0, status, o);
    });
    if (!known) return RF_ERR_BAD_ARG;
    if (bad) return bad;
    RF_LAUNCH_CHECK();
    return 0;
}

}  // extern "C"
