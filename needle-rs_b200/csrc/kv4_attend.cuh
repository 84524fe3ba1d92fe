// What the attention kernels over the paged 4-bit cache share: their
// arguments, the tiles a block of query rows reads, where results go, and the
// joining of a unit's parts.
#pragma once

#include <cfloat>

#include "kv4.cuh"

namespace nd {

struct AttendArgs {
    Kv4Args kv;
    long long q_row, q_head, o_row, o_head;
    FastDiv group;       // query heads a kv head
    FastDiv page_tiles;
    int window, sink, places;
    uint32_t wait_rounds;  // of a wait inside the many-row kernel
    float scale_log2e;
    bool q_vec, o_vec, zero_rest;
    float* parts;   // [runners][2][8 NT * (DV + 2)]; a runner is a warp, for NT = 1 a CTA
    int4* joins;    // [runners]: (sequence, kv head, query block, further runners) of the cut unit that starts there, w < 0: none
};

// The key tiles a block of query rows reads: those of the first `sink`
// positions, then lo .. of the window.
struct Tiles {
    int sink, lo, n;  // n >= 1, so that a block that sees nothing is still written
    __device__ __forceinline__ int at(int i) const { return i < sink ? i : lo + (i - sink); }
};

__device__ __forceinline__ Tiles tiles_of(const AttendArgs& a, long long first, long long last) {
    const int cap = a.kv.max_pages * a.kv.page_tiles * KV4_TILE;  // positions of the table: below 2^31
    const int end = last < 0 ? 0 : (int)min(last, (long long)cap - 1) / KV4_TILE + 1;
    Tiles t;
    t.lo = t.sink = 0;
    if (a.window > 0) {
        t.lo = (int)(min(max(first - a.window + 1, 0LL), (long long)cap)) / KV4_TILE;
        if (a.sink > 0) t.sink = min((min(a.sink, cap) - 1) / KV4_TILE + 1, min(t.lo, end));
    }
    t.n = max(1, t.sink + max(0, end - t.lo));
    return t;
}

struct SeqRows {
    int first, n;    // rows of the call
    long long pos0;  // position of the first
};

__device__ __forceinline__ SeqRows seq_rows(const AttendArgs& a, int s) {
    SeqRows r;
    r.first = kv4_first_row(a.kv, s);
    r.n = max(kv4_first_row(a.kv, s + 1) - r.first, 0);
    r.pos0 = (long long)__ldg(a.kv.lens + s) - r.n;
    return r;
}

// Query rows of a sequence and kv head are numbered token-major: row x is
// head x % group of token x / group. Block b holds 8 NT of them.
template <int NT>
__device__ __forceinline__ Tiles block_tiles(const AttendArgs& a, const SeqRows& r, int b) {
    const int x0 = b * 8 * NT, x1 = min(x0 + 8 * NT, r.n * (int)a.group.d) - 1;
    return tiles_of(a, r.pos0 + a.group(x0), r.pos0 + a.group(x1));
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *(const uint32_t*)&h;
}
__device__ __forceinline__ float2 unpack_half2(uint32_t x) { return __half22float2(*(const __half2*)&x); }
// Codes (in the low four bits of each half; in the next four) to f16 c - 8:
// 1024 + c and 1024 + 16 c are the f16 with those bits under 1024's exponent.
__device__ __forceinline__ uint32_t code_mid(uint32_t x) {
    x |= 0x64006400u;
    uint32_t y;
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(y) : "r"(x), "r"(0xe408e408u));  // -1032
    return y;
}
__device__ __forceinline__ uint32_t code16_mid(uint32_t x) {
    x |= 0x64006400u;
    uint32_t y;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(y) : "r"(x), "r"(0x2c002c00u), "r"(0xd480d480u));  // / 16 - 72
    return y;
}
// Below every score that is not -infinity: the softmax's reference before the
// first key is seen.
constexpr float ATT_LOW = -3.0e38f;
// A row's reference puts its largest weight so far between 2^ATT_TOP and
// 2^(ATT_TOP + 4), just below f16's end: what f16's last step, 2^-24, takes
// from a weight is then 2^-36 of the largest. At 1 instead of 2^11 a key 18
// nats ahead of 32,768 others cost f32 rows 5e-4 of their result.
constexpr float ATT_TOP = 11.f;

// Where query row x of a sequence and kv head has its result.
template <typename T>
struct OutRows {
    T* out;
    const AttendArgs& a;
    int first, h, nrows;
    __device__ __forceinline__ T* at(int x) const {
        const int tok = a.group(x);
        return out + (long long)(first + tok) * a.o_row + (long long)(h * (int)a.group.d + x - tok * (int)a.group.d) * a.o_head;
    }
};

// Output rows behind the last sequence, where the caller wants them zero.
template <int DV, typename T>
__device__ __forceinline__ void zero_rest(const AttendArgs& a, T* out, int wid, int warps, int lane) {
    if (!a.zero_rest || !a.kv.start) return;
    for (int r = kv4_first_row(a.kv, a.kv.seqs) + wid; r < a.kv.rows; r += warps)
        for (int hq = 0; hq < a.kv.heads * (int)a.group.d; hq++)
            for (int d = lane; d < DV; d += 32) out[r * a.o_row + hq * a.o_head + d] = (T)0.f;
}

// out = sum_w 2^(M_w - M) acc_w / sum_w 2^(M_w - M) l_w over the runners w
// that share a unit, in their order. A CTA per runner of the first kernel;
// those where no cut unit starts return at once.
template <int DV, int NT, typename T>
__global__ void __launch_bounds__(512) kv4_join_kernel(AttendArgs a, T* __restrict__ out) {
    constexpr int PART = 8 * NT * (DV + 2), LANES = DV / 4, ROWS = 512 / LANES;  // four dimensions a thread
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    const int4 job = a.joins[blockIdx.x];
    if (job.w < 0) return;
    const SeqRows rows = seq_rows(a, job.x);
    const OutRows<T> to{out, a, rows.first, job.y, rows.n * (int)a.group.d};
    const float* part = a.parts + (size_t)blockIdx.x * 2 * PART;
    const int d = threadIdx.x % LANES * 4;
    for (int y = blockIdx.y * ROWS + threadIdx.x / LANES; y < 8 * NT; y += gridDim.y * ROWS) {
        const int x = job.z * 8 * NT + y;
        if (x >= to.nrows) return;
        // the starting runner's second slot, then the first slot of each further one
        const float* p0 = part + PART;
        float M = p0[8 * NT * DV + y];
#pragma unroll 4
        for (int i = 1; i <= job.w; i++) M = fmaxf(M, part[(size_t)i * 2 * PART + 8 * NT * DV + y]);
        const float r0 = ex2(p0[8 * NT * DV + y] - M);
        float l = p0[8 * NT * (DV + 1) + y] * r0;
        float4 v = *(const float4*)(p0 + y * DV + d);
        v.x *= r0, v.y *= r0, v.z *= r0, v.w *= r0;
#pragma unroll 4
        for (int i = 1; i <= job.w; i++) {
            const float* p = part + (size_t)i * 2 * PART;
            const float r = ex2(p[8 * NT * DV + y] - M);
            const float4 u = *(const float4*)(p + y * DV + d);
            l = __fmaf_rn(p[8 * NT * (DV + 1) + y], r, l);
            v.x = __fmaf_rn(u.x, r, v.x), v.y = __fmaf_rn(u.y, r, v.y), v.z = __fmaf_rn(u.z, r, v.z), v.w = __fmaf_rn(u.w, r, v.w);
        }
        const float norm = l == 0.f ? 0.f : 1.f / l;
        T* o = to.at(x) + d;
        o[0] = (T)(v.x * norm), o[1] = (T)(v.y * norm), o[2] = (T)(v.z * norm), o[3] = (T)(v.w * norm);
    }
}

// The tcgen05 kernel for long runs of query rows (kv4_prefill.cu): rows a
// unit, workspace and launch. `dk` chooses the head dimensions; 16-bit types.
constexpr int PRE_ROWS = 256;
size_t prefill_ws_bytes(int dv, int* ctas);
void prefill_launch(const AttendArgs& a, int dk, int type, const void* q, void* out, void* ws, cudaStream_t st);

}  // namespace nd
