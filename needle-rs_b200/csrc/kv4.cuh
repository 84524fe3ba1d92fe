// The paged 4-bit key/value cache: its layout, the arguments its kernels
// share, and how a row of new tokens finds its sequence and its place.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace nd {

// A tile is 16 positions of one kv head, contiguous: key codes [16][dk / 2],
// value codes [16][dv / 2], then the keys' and the values' f16 (scale,
// minimum) pairs [16] each. Two codes a byte, the lower dimension in the low
// nibble; value = minimum + scale * code. A page holds its heads one after
// another, page / 16 tiles each. Sixteen positions are one m16 operand of the
// tensor cores, so a tile is what a warp loads and multiplies at a time,
// whatever the page size.
constexpr int KV4_TILE = 16;
__host__ __device__ constexpr int kv4_tile_bytes(int dk, int dv) { return KV4_TILE * (dk / 2 + dv / 2 + 8); }

struct Kv4Args {
    uint8_t* pool;
    long long page_stride;  // bytes
    const int32_t* table;
    int table_stride, max_pages, num_pages;
    int page_tiles;  // tiles a page and head
    int heads, seqs, rows;
    const int32_t* lens;
    const int32_t* start;  // NULL: rows / seqs rows each
};

// First row of sequence s, kept inside [0, rows] whatever `start` holds.
__device__ __forceinline__ int kv4_first_row(const Kv4Args& a, int s) {
    if (!a.start) return (int)((long long)s * (a.rows / a.seqs));
    return min(max(__ldg(a.start + s), 0), a.rows);
}

// The sequence of row r: how many of the sequences end at or before it,
// found by the whole warp 32 ends at a time. False for a row behind the last
// sequence (or outside its own where `start` does not ascend).
__device__ __forceinline__ bool kv4_find_row(const Kv4Args& a, int r, int lane, int* seq, int* first, int* n) {
    int s;
    if (!a.start) {
        s = r / (a.rows / a.seqs);
    } else {
        int lo = 0, size = a.seqs;
        while (size > 0) {
            const int step = (size + 31) / 32, at = lane * step + step - 1;
            const bool before = at < size && __ldg(a.start + 1 + lo + at) <= r;
            const int c = __popc(__ballot_sync(0xffffffffu, before));
            lo += c * step;
            size = min(step - 1, size - c * step);
        }
        s = lo;
    }
    if (s >= a.seqs) return false;
    const int b = kv4_first_row(a, s), e = kv4_first_row(a, s + 1);
    *seq = s;
    *first = b;
    *n = e - b;
    return r >= b && r < e;
}

// The tile that holds position pos of sequence s for head 0, or NULL where
// the table has no page of the pool for it.
__device__ __forceinline__ uint8_t* kv4_tile_of(const Kv4Args& a, int s, long long pos, int tile_bytes) {
    const long long tile = pos / KV4_TILE;
    if (pos < 0 || tile >= (long long)a.max_pages * a.page_tiles) return nullptr;
    const int page = __ldg(a.table + (size_t)s * a.table_stride + tile / a.page_tiles);
    if (page < 0 || page >= a.num_pages) return nullptr;
    return a.pool + (size_t)page * a.page_stride + (size_t)(tile % a.page_tiles) * tile_bytes;
}

// n / d for 0 <= n < 2^31 by a multiplication.
struct FastDiv {
    uint32_t d, mul, shift;
    FastDiv(uint32_t x = 1) : d(x), mul(0), shift(0) {
        while ((1ull << shift) < d) shift++;
        mul = (uint32_t)((((1ull << shift) - d) << 32) / d + 1);
    }
    __device__ __forceinline__ int operator()(int n) const { return (int)((__umulhi((uint32_t)n, mul) + (uint32_t)n) >> shift); }
};

// Two f32 operations in one instruction.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pair(float a, float b) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpair(f32x2 x) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
    return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// Eight consecutive values as floats, by 16-byte loads where `vec`.
__device__ __forceinline__ void load8(const float* p, bool vec, float* v) {
    if (vec) {
        const float4 a = __ldg((const float4*)p), b = __ldg((const float4*)p + 1);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = __ldg(p + i);
    }
}
__device__ __forceinline__ void load8(const __half* p, bool vec, float* v) {
    if (vec) {
        const uint4 a = __ldg((const uint4*)p);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = __half22float2(*(const __half2*)&w[i]);
            v[2 * i] = f.x, v[2 * i + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = __half2float(p[i]);
    }
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, bool vec, float* v) {
    if (vec) {
        const uint4 a = __ldg((const uint4*)p);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; i++) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = __bfloat162float(p[i]);
    }
}

// Eight floats rounded once to the row's type, by 16-byte stores where `vec`.
__device__ __forceinline__ void store8(float* p, bool vec, const float* v) {
    if (vec) {
        ((float4*)p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        ((float4*)p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) p[i] = v[i];
    }
}
__device__ __forceinline__ void store8(__half* p, bool vec, const float* v) {
    if (vec) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
            w[i] = *(const uint32_t*)&h;
        }
        *(uint4*)p = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) p[i] = __float2half_rn(v[i]);
    }
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, bool vec, const float* v) {
    if (vec) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
            w[i] = *(const uint32_t*)&h;
        }
        *(uint4*)p = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) p[i] = __float2bfloat16_rn(v[i]);
    }
}

}  // namespace nd
