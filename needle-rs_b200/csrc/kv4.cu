// Rows into and out of the paged 4-bit cache (nd_op_kv4_append,
// nd_op_kv4_read). A row of values x (one position, one kv head, its key or
// its value) is kept as codes c in 0 .. 15 with an f16 scale s and minimum m,
// x ~ m + s c; every step is an IEEE f32 operation rounded once, so codes do
// not depend on how the work is split.

#include <cfloat>
#include <stdexcept>
#include <string>

#include "kernels.h"
#include "kv4.cuh"
#include "kv4_host.h"

namespace nd {

// A warp takes one row of the call: its 2 * heads vectors, L lanes each with
// sixteen values a lane (so a lane forms 64 bits of codes), 32 / L vectors at
// a time. Bound by instructions, not by HBM: a vector costs about as many for
// its minimum, its place and its parameters as for its codes, which is why a
// lane has sixteen values and not the eight of one load (12,000 rows of 8
// heads of 128 bf16, in and out again: 45 us, with eight 50). The search for
// the row's sequence costs two or three dependent loads of a warp, not
// log2(seqs), and the first values are on their way meanwhile.
template <int DK, int DV>
struct RowSplit {
    static constexpr int L = DK > 64 || DV > 64 ? 8 : 4;
    static constexpr int PER = 32 / L;
};

constexpr int ROW_WARPS = 8;

// Sixteen values to codes, given their row's scale and minimum. A code is the
// nearest whole number to the f32 quotient of d = x - m by s. By a reciprocal
// the quotient is off by 2^-21 of it at most: its nearest whole number r is
// the right one unless d lies near the middle between two, |d - r s| near s /
// 2 (or r was cut to 0 or 15), and those are divided out. Adding 1.5 * 2^23
// rounds to a whole number that the low bits hold.
__device__ __forceinline__ uint2 codes_of(const float* x, float sf, float mf) {
    if (!(sf > 0.f)) return make_uint2(0, 0);  // all values alike, or no numbers
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(sf));
    const f32x2 m2 = pair(-mf, -mf), inv2 = pair(inv, inv), s2 = pair(-sf, -sf);
    const f32x2 up = pair(12582912.f, 12582912.f), down = pair(-12582912.f, -12582912.f);
    float off = 0.f;
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
        const f32x2 d = add2(pair(x[i], x[i + 1]), m2);
        float2 y = unpair(mul2(d, inv2));
        y.x = fminf(fmaxf(y.x, 0.f), 15.f), y.y = fminf(fmaxf(y.y, 0.f), 15.f);
        const f32x2 t = add2(pair(y.x, y.y), up);
        const float2 e = unpair(fma2(add2(t, down), s2, d)), f = unpair(t);
        off = fmaxf(off, fmaxf(fabsf(e.x), fabsf(e.y)));
        w[i / 8] += (__float_as_uint(f.x) << (4 * (i % 8))) + (__float_as_uint(f.y) << (4 * (i % 8) + 4));
    }
    w[0] -= 0x4b400000u * 0x11111111u, w[1] -= 0x4b400000u * 0x11111111u;  // the constants
    if (__builtin_expect(!(off < 0.4999f * sf), 0)) {
        w[0] = w[1] = 0;
#pragma unroll
        for (int i = 0; i < 16; i++)
            w[i / 8] |= (uint32_t)(int)fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(x[i], mf), sf)), 0.f), 15.f) << (4 * (i % 8));
    }
    return make_uint2(w[0], w[1]);
}

template <int DK, int DV, typename T>
__global__ void __launch_bounds__(32 * ROW_WARPS) kv4_append_kernel(Kv4Args a, const T* __restrict__ k, long long k_row, long long k_head,
                                                                    const T* __restrict__ v, long long v_row, long long v_head, bool vec) {
    constexpr int TB = kv4_tile_bytes(DK, DV), L = RowSplit<DK, DV>::L, PER = RowSplit<DK, DV>::PER;
    const int lane = threadIdx.x & 31, r = blockIdx.x * ROW_WARPS + (threadIdx.x >> 5);
    if (r >= a.rows) return;
    const int sub = lane % L, d0 = 16 * sub, step = gridDim.y * PER;
    int j = blockIdx.y * PER + lane / L;
    float x[16];
    auto fetch = [&]() {
        const bool val = j >= a.heads;
        if (j >= 2 * a.heads || d0 >= (val ? DV : DK)) return;
        const T* p = val ? v + r * v_row + (j - a.heads) * v_head + d0 : k + r * k_row + j * k_head + d0;
        load8(p, vec, x);
        load8(p + 8, vec, x + 8);
    };
    fetch();
    int s, first, n;
    if (!kv4_find_row(a, r, lane, &s, &first, &n)) return;
    const long long pos = (long long)__ldg(a.lens + s) - n + (r - first);
    uint8_t* tile0 = kv4_tile_of(a, s, pos, TB);
    if (!tile0) return;
    const int slot = (int)(pos % KV4_TILE);
    while (true) {
        const bool val = j >= a.heads;
        const int h = val ? j - a.heads : j, D = val ? DV : DK;
        const bool on = j < 2 * a.heads && d0 < D;
        float lo = FLT_MAX, hi = -FLT_MAX;
        bool bad = false;
        if (on) {
            f32x2 zero = 0;  // NaN where a value is not finite
#pragma unroll
            for (int i = 0; i < 16; i += 2) zero = fma2(pair(x[i], x[i + 1]), 0, zero);
#pragma unroll
            for (int i = 0; i < 16; i++) lo = fminf(lo, x[i]), hi = fmaxf(hi, x[i]);
            const float2 z = unpair(zero);
            bad = !(z.x == 0.f && z.y == 0.f);
        }
#pragma unroll
        for (int o = 1; o < L; o *= 2) {
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        }
        bad = (__ballot_sync(0xffffffffu, bad) >> (lane & ~(L - 1)) & ((1u << L) - 1)) != 0;
        if (on) {
            __half sh = __float2half_rn(fminf(__fdiv_rn(__fsub_rn(hi, lo), 15.0f), 65504.0f));
            __half mh = __float2half_rn(fminf(fmaxf(lo, -65504.0f), 65504.0f));
            if (bad) sh = mh = __ushort_as_half(0x7fff);
            const uint2 w = codes_of(x, __half2float(sh), __half2float(mh));
            uint8_t* t = tile0 + (size_t)h * a.page_tiles * TB;
            *(uint2*)(t + (val ? 8 * DK : 0) + slot * (D / 2) + 8 * sub) = w;
            if (sub == 0) *(__half2*)(t + 8 * (DK + DV) + (val ? 64 : 0) + 4 * slot) = __halves2half2(sh, mh);
        }
        j += step;
        if (j - lane / L >= 2 * a.heads) break;
        fetch();
    }
}

template <int DK, int DV, typename T>
__global__ void __launch_bounds__(32 * ROW_WARPS) kv4_read_kernel(Kv4Args a, T* __restrict__ k, long long k_row, long long k_head,
                                                                  T* __restrict__ v, long long v_row, long long v_head, bool vec, bool zero_rest) {
    constexpr int TB = kv4_tile_bytes(DK, DV), L = RowSplit<DK, DV>::L, PER = RowSplit<DK, DV>::PER;
    const int lane = threadIdx.x & 31, r = blockIdx.x * ROW_WARPS + (threadIdx.x >> 5);
    if (r >= a.rows) return;
    int s, first, n;
    long long pos = 0;
    const uint8_t* tile0 = nullptr;
    if (kv4_find_row(a, r, lane, &s, &first, &n)) {
        pos = (long long)__ldg(a.lens + s) - n + (r - first);
        tile0 = kv4_tile_of(a, s, pos, TB);
    } else if (!zero_rest) {
        return;
    }
    const int slot = (int)(pos % KV4_TILE), sub = lane % L, d0 = 16 * sub;
#pragma unroll 2
    for (int j = blockIdx.y * PER + lane / L; j < 2 * a.heads; j += gridDim.y * PER) {
        const bool val = j >= a.heads;
        const int h = val ? j - a.heads : j, D = val ? DV : DK;
        if (d0 >= D) continue;
        uint2 w = make_uint2(0, 0);  // no such position: zeros
        float2 sm = make_float2(0.f, 0.f);
        if (tile0) {
            const uint8_t* t = tile0 + (size_t)h * a.page_tiles * TB;
            w = *(const uint2*)(t + (val ? 8 * DK : 0) + slot * (D / 2) + 8 * sub);
            sm = __half22float2(*(const __half2*)(t + 8 * (DK + DV) + (val ? 64 : 0) + 4 * slot));
        }
        float x[16];
        // 2^23 + c has the code in its low bits; the product of an f16 and a
        // code is exact: one rounding
        const f32x2 s2 = pair(sm.x, sm.x), m2 = pair(sm.y, sm.y), down = pair(-8388608.f, -8388608.f);
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
            const uint32_t c = (i < 8 ? w.x : w.y) >> (4 * (i % 8));
            const f32x2 f = add2(pair(__uint_as_float((c & 15) | 0x4b000000u), __uint_as_float((c >> 4 & 15) | 0x4b000000u)), down);
            const float2 y = unpair(fma2(s2, f, m2));
            x[i] = y.x, x[i + 1] = y.y;
        }
        T* p = val ? v + r * v_row + h * v_head + d0 : k + r * k_row + h * k_head + d0;
        store8(p, vec, x);
        store8(p + 8, vec, x + 8);
    }
}

Kv4Args kv4_args(const nd_kv4* kv, const char* what) {
    auto fail = [&](const std::string& m) { throw std::runtime_error(std::string(what) + ": " + m); };
    if (!kv) fail("null cache");
    if (!kv->pool || !kv->table || !kv->lens) fail("null pointer");
    if (kv->num_pages < 1 || kv->heads < 1 || kv->max_pages < 1 || kv->seqs < 1 || kv->rows < 0) fail("sizes must be positive");
    if (kv->heads > 65535 || kv->seqs > (1 << 20)) fail("at most 65535 heads and 2^20 sequences");
    if (kv->page < 16 || kv->page % 16) fail("page must be a multiple of 16 positions");
    if (!((kv->dk == 48 && kv->dv == 64) || (kv->dk == 64 && kv->dv == 64) || (kv->dk == 128 && kv->dv == 128)))
        fail("(dk, dv) must be (48, 64), (64, 64) or (128, 128)");
    if (kv->table_stride < kv->max_pages) fail("table rows overlap");
    if ((uintptr_t)kv->pool % 16 || kv->page_stride % 16) fail("the pool and its page stride must be 16-byte aligned");
    const long long bytes = (long long)kv->heads * (kv->page / 16) * kv4_tile_bytes(kv->dk, kv->dv);
    if (kv->page_stride < bytes) fail("pages overlap");
    if ((long long)kv->max_pages * kv->page > 0x7fffffffLL) fail("more than 2^31 - 1 positions a sequence");
    if (!kv->start && kv->rows % kv->seqs) fail("without start, rows must be a multiple of the sequences");
    return Kv4Args{(uint8_t*)kv->pool, kv->page_stride, kv->table,   kv->table_stride, kv->max_pages, kv->num_pages,
                   kv->page / 16,      kv->heads,       kv->seqs,    kv->rows,         kv->lens,      kv->start};
}

bool kv4_vec(int type, const void* p, long long row, long long head) {
    const int e = type == ND_F32 ? 4 : 2;
    return (uintptr_t)p % 16 == 0 && row * e % 16 == 0 && head * e % 16 == 0;
}

void kv4_check_rows(const char* what, int type, const void* p, long long row, long long head) {
    auto fail = [&](const std::string& m) { throw std::runtime_error(std::string(what) + ": " + m); };
    if (type != ND_F32 && type != ND_F16 && type != ND_BF16) fail("unknown type");
    if (!p) fail("null pointer");
    if ((uintptr_t)p % (type == ND_F32 ? 4 : 2)) fail("rows must be aligned to their type");
    if (row < 0 || head < 0) fail("negative strides");
}

// Rows that are written may not share memory.
static void check_distinct(const char* what, long long row, long long head, int rows, int heads, int d) {
    const bool row_major = head >= d && (rows <= 1 || row >= (long long)(heads - 1) * head + d);
    const bool head_major = row >= d && (heads <= 1 || head >= (long long)(rows - 1) * row + d);
    const bool one = heads == 1 && (rows <= 1 || row >= d);
    if (!row_major && !head_major && !one) throw std::runtime_error(std::string(what) + ": output rows overlap");
}

void kv4_check_out(const char* what, int type, const void* p, long long row, long long head, int rows, int heads, int d) {
    kv4_check_rows(what, type, p, row, head);
    check_distinct(what, row, head, rows, heads, d);
}

// Calls f with the cache's head dimensions and the rows' type as templates.
template <typename F>
static void dispatch(int dk, int type, F&& f) {
    auto typed = [&](auto dkc, auto dvc) {
        if (type == ND_F32) f(dkc, dvc, (float*)nullptr);
        else if (type == ND_F16) f(dkc, dvc, (__half*)nullptr);
        else f(dkc, dvc, (__nv_bfloat16*)nullptr);
    };
    if (dk == 48) typed(std::integral_constant<int, 48>(), std::integral_constant<int, 64>());
    else if (dk == 64) typed(std::integral_constant<int, 64>(), std::integral_constant<int, 64>());
    else typed(std::integral_constant<int, 128>(), std::integral_constant<int, 128>());
}

// Rows go eight to a CTA; with few rows the vectors of a row are spread over
// grid.y so that a handful of rows of many heads still fills the GPU.
static dim3 row_grid(const Kv4Args& a, int per) {
    const int x = (a.rows + ROW_WARPS - 1) / ROW_WARPS, steps = (2 * a.heads + per - 1) / per;
    const int want = (4 * device_sm_count() + x - 1) / x;
    return dim3(x, std::min(std::min(steps, std::max(want, 1)), 65535));
}

}  // namespace nd

using namespace nd;

extern "C" {

int nd_op_kv4_append(const nd_kv4* kv, int type, const void* k, long long k_row, long long k_head, const void* v,
                     long long v_row, long long v_head, void* stream) {
    return op_call([&] {
        const char* what = "nd_op_kv4_append";
        const Kv4Args a = kv4_args(kv, what);
        if (a.rows == 0) return;
        kv4_check_rows(what, type, k, k_row, k_head);
        kv4_check_rows(what, type, v, v_row, v_head);
        const bool vec = kv4_vec(type, k, k_row, k_head) && kv4_vec(type, v, v_row, v_head);
        OnDevice on(kv->device, what);
        dispatch(kv->dk, type, [&](auto dk, auto dv, auto* t) {
            using T = std::remove_pointer_t<decltype(t)>;
            constexpr int DK = decltype(dk)::value, DV = decltype(dv)::value;
            kv4_append_kernel<DK, DV, T><<<row_grid(a, RowSplit<DK, DV>::PER), 32 * ROW_WARPS, 0, (cudaStream_t)stream>>>(
                a, (const T*)k, k_row, k_head, (const T*)v, v_row, v_head, vec);
        });
        op_launched(what);
    });
}

int nd_op_kv4_read(const nd_kv4* kv, int type, void* k, long long k_row, long long k_head, void* v, long long v_row,
                   long long v_head, int flags, void* stream) {
    return op_call([&] {
        const char* what = "nd_op_kv4_read";
        const Kv4Args a = kv4_args(kv, what);
        if (flags & ~ND_ZERO_REST) throw std::runtime_error("nd_op_kv4_read: unknown flags");
        if (a.rows == 0) return;
        kv4_check_out(what, type, k, k_row, k_head, a.rows, a.heads, kv->dk);
        kv4_check_out(what, type, v, v_row, v_head, a.rows, a.heads, kv->dv);
        const bool vec = kv4_vec(type, k, k_row, k_head) && kv4_vec(type, v, v_row, v_head);
        OnDevice on(kv->device, what);
        dispatch(kv->dk, type, [&](auto dk, auto dv, auto* t) {
            using T = std::remove_pointer_t<decltype(t)>;
            constexpr int DK = decltype(dk)::value, DV = decltype(dv)::value;
            kv4_read_kernel<DK, DV, T><<<row_grid(a, RowSplit<DK, DV>::PER), 32 * ROW_WARPS, 0, (cudaStream_t)stream>>>(
                a, (T*)k, k_row, k_head, (T*)v, v_row, v_head, vec, flags & ND_ZERO_REST);
        });
        op_launched(what);
    });
}

}  // extern "C"
