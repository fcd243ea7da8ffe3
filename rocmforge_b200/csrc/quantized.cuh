// What the kernels with 4-bit weights share: the stored form, asynchronous copies, the output.
//
// How weights are stored.  The unit is a tile of 16 rows by 64 columns, 512 bytes in a row, the tiles of 16 rows one after another along
// K.  The 16 bytes of lane 4 g + t hold rows g and g + 8 of the columns 32 c + 8 t .. + 7, c = 0, 1, as four words (row g: c = 0, 1; row
// g + 8: c = 0, 1); the low half of byte b of a word is column b of the eight, the high half column 4 + b.  So a lane's one 16-byte load
// is what it feeds to two mma.m16n8k32 of 8-bit integers (or four m16n8k16 of bfloat16 numbers): halves of bytes become operands with
// one shift and one mask, in place, and a row's 8 numbers for the same columns are one 8-byte load of the row as it lies.  The scales
// lie beside them, [tile of rows, group, 16], row g + 8 r at 2 g + r: the two that a lane needs are one word.
#pragma once
#include "common.cuh"

__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool there) {       // zeros if it is not there
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t to, const void* from, bool there) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(there ? 4 : 0) : "memory");
}
// ... by the lanes with `mine` alone (a predicate, no branch: the warp stays together for the matrix instructions behind it)
__device__ __forceinline__ void copy4_if(uint32_t to, const void* from, bool there, bool mine) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.u32 p, %3, 0;\n\t"
        "@p cp.async.ca.shared.global [%0], [%1], 4, %2;\n\t}"
        ::"r"(to), "l"(from), "r"(there ? 4 : 0), "r"((uint32_t)mine) : "memory");
}

struct W4Out {
    void* out;               // [M, N] float32 if is_f32, else bfloat16; add: float32, added into
    const void* bias;        // [N] or null
    int bias_is_f32, is_f32, add, M, N;
    int fours;               // four neighbours of a row lie together on a boundary of their size
};
__device__ __forceinline__ void w4_write(const W4Out& o, int t, int n, float v) {
    if (n >= o.N) return;
    if (o.bias != nullptr) v += load_vec(o.bias, o.bias_is_f32, n);
    const size_t at = (size_t)t * o.N + n;
    if (o.add) reinterpret_cast<float*>(o.out)[at] += v;
    else if (o.is_f32) reinterpret_cast<float*>(o.out)[at] = v;
    else reinterpret_cast<__nv_bfloat16*>(o.out)[at] = __float2bfloat16_rn(v);
}
// Columns n .. n + 3, n a multiple of 4.  (What is read is read before anything is written: a load behind a store would wait for it.)
__device__ __forceinline__ void w4_write4(const W4Out& o, int t, int n, float4 v4) {
    if (n >= o.N) return;
    const int live = min(4, o.N - n);
    float v[4] = {v4.x, v4.y, v4.z, v4.w};
    float* to = reinterpret_cast<float*>(o.out) + (size_t)t * o.N + n;   // (32-bit results)
    if (o.bias != nullptr) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < live) v[j] += load_vec(o.bias, o.bias_is_f32, n + j);
    }
    if (o.add) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < live) v[j] += to[j];
    }
    if (o.fours && o.is_f32) {
        *reinterpret_cast<float4*>(to) = make_float4(v[0], v[1], v[2], v[3]);
    } else if (o.is_f32) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < live) to[j] = v[j];
    } else {
        __nv_bfloat16* to16 = reinterpret_cast<__nv_bfloat16*>(o.out) + (size_t)t * o.N + n;
        if (o.fours) {
            const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
            *reinterpret_cast<uint2*>(to16) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j < live) to16[j] = __float2bfloat16_rn(v[j]);
        }
    }
}

static bool bad_group(int G) { return G != 32 && G != 64 && G != 128; }
static int padded(int K, int G) { const int u = G > 64 ? G : 64; return (K + u - 1) / u * u; }
static bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
static W4Out w4_out(void* out, const void* bias, int bias_is_f32, int is_f32, int add, int M, int N) {
    return {out, bias, bias_is_f32, is_f32, add, M, N, N % 4 == 0 && aligned(out, is_f32 ? 16 : 8)};
}
