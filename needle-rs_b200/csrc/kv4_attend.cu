// Attention over the paged 4-bit cache (nd_op_kv4_attend).
//
// With k_j = mk_j + sk_j c_j and v_j = mv_j + sv_j e_j (c, e the codes, one
// f16 scale and minimum a row of values):
//   q.k_j = sk_j (q.c_j) + mk_j sum(q)
//   out   = (sum_j (p_j sv_j) e_j + sum_j p_j mv_j) / sum_j p_j,
// so the codes go to the tensor cores as they are and the cache is never
// dequantized. A warp takes 16 positions at a time (mma.sync m16n8k16, f16
// in, f32 sums), the positions (or value dimensions) as M and 8 * NT query
// rows of one kv head as N: with few queries a row, as in decoding, that
// wastes half of what queries-as-M would.
//
// Codes as f16 operands: a code in the low four bits of a half is the
// subnormal c * 2^-24, exact, so one AND makes two operands; the next four
// bits make 16 c * 2^-24, whose 16 is taken out of the matching query value
// beforehand (q is scaled per row by a power of two so that its f16 keeps it)
// or out of the accumulator row afterwards. 2^24 is put back in f32.
// Weights p sv are split into two f16 terms (22 bits) for f32 and f16 rows;
// bf16 rows take one: its 2^-12 is far below the output's own 2^-9.
//
// f32 rows. The tensor cores truncate their sums near the 24th bit, and codes
// counted from the minimum add up to much more than the result, so what is
// enough for 16-bit outputs loses f32's last bits twice over. For f32:
// - q is split in fixed point: q = q1 + q2 with 11 bits each below the row's
//   largest value (2^-24 of it is left). A k-sum of codes times either term,
//   started at -8 sum(q_i) so that codes count from the middle, stays below
//   2^24 units: it is exact, whatever the order.
// - value codes are made the f16 e - 8 (one more instruction a pair), each
//   tile's sum starts at zero and is added to the accumulator rounded.
// Measured: 5e-7 of the result against 64 bits where the plain way had 4e-5
// (keys and values with outlying channels).
//
// A warp keeps the softmax's running reference M per query row (a power-of-
// two argument: scores carry log2 e) and rescales only when a new exponent
// passes it by more than 4, since only the quotient counts. The reference is
// taken over score + log2 sv, so that the f16 weight p sv is at most 16
// whatever the values' scale.
//
// Work split: the tiles of all (sequence, kv head, query block) units are one
// list, each warp takes an equal run of it, whatever the lengths; every CTA
// finds its place by summing the sequences' tile counts itself. A unit cut by
// a run's border leaves unnormalised parts in the workspace, joined by a
// second kernel in a fixed order.

#include <cfloat>
#include <cstring>

#include "kernels.h"
#include "kv4.cuh"
#include "kv4_host.h"

namespace nd {

constexpr int ATT_WARPS = 4, ATT_STAGES = 4;
constexpr int ATT_MIN_SHARE = 4;  // tiles: a shorter run costs more to join than it takes

struct AttendArgs {
    Kv4Args kv;
    long long q_row, q_head, o_row, o_head;
    int group;  // query heads a kv head
    int window, sink;
    float scale_log2e;
    int q_vec, o_vec;
    float* parts;   // [warps][2][8 NT * (DV + 2)]
    int4* joins;    // [warps]: (sequence, kv head, query block, further warps) of the cut unit that starts there, w < 0: none
};

// The key tiles a block of query rows reads: those of the first `sink`
// positions, then lo .. hi of the window.
struct Tiles {
    int sink, lo, n;  // n >= 1, so that a block that sees nothing is still written
    __device__ __forceinline__ int at(int i) const { return i < sink ? i : lo + (i - sink); }
};

__device__ __forceinline__ Tiles tiles_of(const AttendArgs& a, long long first, long long last) {
    const long long cap = (long long)a.kv.max_pages * a.kv.page_tiles * KV4_TILE;
    const long long hi = min(last, cap - 1);
    long long lo = a.window > 0 ? max(first - a.window + 1, 0LL) : 0LL;
    Tiles t;
    t.lo = (int)(min(lo, cap) / KV4_TILE);
    const int end = hi < 0 ? 0 : (int)(hi / KV4_TILE) + 1;
    int sink = 0;
    if (a.window > 0 && a.sink > 0) sink = min((int)((min((long long)a.sink, cap) + KV4_TILE - 1) / KV4_TILE), min(t.lo, end));
    t.sink = sink;
    t.n = max(1, sink + max(0, end - t.lo));
    return t;
}

struct SeqRows {
    int first, n;        // rows of the call
    long long pos0;      // position of the first
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
    const int x0 = b * 8 * NT, x1 = min(x0 + 8 * NT, r.n * a.group) - 1;
    return tiles_of(a, r.pos0 + x0 / a.group, r.pos0 + x1 / a.group);
}

template <int NT>
__device__ __forceinline__ long long seq_tiles(const AttendArgs& a, const SeqRows& r) {
    const int blocks = (r.n * a.group + 8 * NT - 1) / (8 * NT);
    long long t = 0;
    for (int b = 0; b < blocks; b++) t += block_tiles<NT>(a, r, b).n;
    return t;
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
__device__ __forceinline__ void mma16816(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
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
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src) : "memory");
}

template <int DK, int DV, int NT, typename T>
struct AttendShape {
    static constexpr int TB = kv4_tile_bytes(DK, DV);
    static constexpr int QS = std::is_same<T, float>::value ? 2 : 1;           // f16 terms of a query value
    static constexpr int WS = std::is_same<T, __nv_bfloat16>::value ? 1 : 2;  // f16 terms of a weight
    static constexpr int KSTEPS = DK / 16;
    static constexpr int QREGS = KSTEPS * 2 * QS;                 // a query block's operands, per 8 rows
    static constexpr bool Q_SMEM = NT * QREGS > 32;               // else they stay in registers
    static constexpr int SMEM = ATT_WARPS * (ATT_STAGES * TB + (Q_SMEM ? NT * QREGS * 128 : 0));
    static constexpr int CTAS = NT == 1 ? 4 : NT == 2 ? 3 : 2;
    static constexpr int PART = 8 * NT * (DV + 2);                // floats
};

template <int DK, int DV, int NT, typename T>
__global__ void __launch_bounds__(32 * ATT_WARPS, AttendShape<DK, DV, NT, T>::CTAS)
    kv4_attend_kernel(AttendArgs a, const T* __restrict__ q, T* __restrict__ out) {
    using Sh = AttendShape<DK, DV, NT, T>;
    constexpr int TB = Sh::TB, QS = Sh::QS, WS = Sh::WS, KS = Sh::KSTEPS, MT = DV / 16, VW = DV / 64;
    constexpr bool MID = std::is_same<T, float>::value;  // codes count from 8
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ long long sums[32 * ATT_WARPS + 1];
    __shared__ long long warp_sums[ATT_WARPS];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
    const int H = a.kv.heads, S = a.kv.seqs;

    // the list's length, and its prefix at every chunk of `per` sequences
    const int per = (S + 32 * ATT_WARPS - 1) / (32 * ATT_WARPS);
    {
        long long mine = 0;
        for (int s = tid * per; s < min((tid + 1) * per, S); s++) mine += seq_tiles<NT>(a, seq_rows(a, s)) * H;
        long long incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const long long up = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += up;
        }
        if (lane == 31) warp_sums[warp] = incl;
        __syncthreads();
        for (int w = 0; w < warp; w++) incl += warp_sums[w];
        sums[tid + 1] = incl;
        if (tid == 0) sums[0] = 0;
        __syncthreads();
    }
    const long long total = sums[32 * ATT_WARPS];
    const int warps = gridDim.x * ATT_WARPS, wid = blockIdx.x * ATT_WARPS + warp;
    const long long share = max((total + warps - 1) / warps, (long long)ATT_MIN_SHARE);
    const long long begin = min(wid * share, total), end = min(begin + share, total);
    if (lane == 0) a.joins[wid] = make_int4(0, 0, 0, -1);
    if (begin >= end) return;

    // the unit at `begin`
    int s;
    {
        int lo = 0, hi = 32 * ATT_WARPS;  // sums[lo] <= begin < sums[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (sums[mid] <= begin) lo = mid;
            else hi = mid;
        }
        s = lo * per;
        hi = lo;
    }
    long long rem = begin - sums[s / per];
    SeqRows rows = seq_rows(a, s);
    long long per_head = seq_tiles<NT>(a, rows);
    while (rem >= per_head * H) {
        rem -= per_head * H;
        rows = seq_rows(a, ++s);
        per_head = seq_tiles<NT>(a, rows);
    }
    int h = (int)(rem / per_head), b = 0;
    rem -= h * per_head;
    Tiles tl = block_tiles<NT>(a, rows, 0);
    while (rem >= tl.n) {
        rem -= tl.n;
        tl = block_tiles<NT>(a, rows, ++b);
    }
    int off = (int)rem;

    uint8_t* ring = smem + warp * ATT_STAGES * TB;
    const uint32_t ring_s = (uint32_t)__cvta_generic_to_shared(ring);
    uint32_t* qsm = (uint32_t*)(smem + ATT_WARPS * ATT_STAGES * TB) + warp * (NT * Sh::QREGS * 32) + lane;
    const size_t head_stride = (size_t)a.kv.page_tiles * TB;

    long long cur = begin;
    while (true) {
        const int m = (int)min((long long)(tl.n - off), end - cur);
        const int nrows = rows.n * a.group;

        // page ids of the next tiles, 32 at a time, one batch ahead
        const int32_t* trow = a.kv.table + (size_t)s * a.kv.table_stride;
        const int i_end = off + m;
        auto fetch_page = [&](int i) {
            const int t = i < i_end ? tl.at(i) / a.kv.page_tiles : 0;
            return i < i_end && t < a.kv.max_pages ? __ldg(trow + t) : -1;
        };
        int ids = fetch_page(off + lane), ids_next = fetch_page(off + 32 + lane);
        uint32_t okbits = 0;  // by stage: the tile's page exists
        int issued = 0;
        auto issue = [&]() {
            if (issued < m) {
                const int i = off + issued, page = __shfl_sync(0xffffffffu, ids, issued & 31);
                const bool ok = page >= 0 && page < a.kv.num_pages;
                const int st = issued % ATT_STAGES;
                okbits = (okbits & ~(1u << st)) | ((uint32_t)ok << st);
                if (ok) {
                    const uint8_t* src = a.kv.pool + (size_t)page * a.kv.page_stride + h * head_stride + (size_t)(tl.at(i) % a.kv.page_tiles) * TB;
#pragma unroll
                    for (int j = 0; j < (TB / 16 + 31) / 32; j++)
                        if (j * 32 + lane < TB / 16) copy16(ring_s + st * TB + (j * 32 + lane) * 16, src + (j * 32 + lane) * 16);
                }
                issued++;
                if ((issued & 31) == 0) {
                    ids = ids_next;
                    ids_next = fetch_page(off + issued + 32 + lane);
                }
            }
            asm volatile("cp.async.commit_group;\n" ::: "memory");
        };
        __syncwarp();  // the ring's last tile has been read by every lane
#pragma unroll
        for (int i = 0; i < ATT_STAGES - 1; i++) issue();

        // the query block: lane (g, c) holds of query row 8 t + g the
        // dimensions whose codes it will hold of every key
        uint32_t qreg[Sh::Q_SMEM ? 1 : NT * Sh::QREGS];
        float f0[NT][2], f1[NT][2], mid[QS == 2 ? NT : 1][2][2];
        int seen_hi[NT][2];
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const int x = b * 8 * NT + 8 * t + g;
            const bool on = x < nrows;
            float v[DK / 4];
#pragma unroll
            for (int i = 0; i < DK / 4; i++) v[i] = 0.f;
            if (on) {
                const T* p = q + (rows.first + x / a.group) * a.q_row + (h * a.group + x % a.group) * a.q_head;
                if constexpr (DK == 48) {
                    load8(p + 8 * c, a.q_vec, v);
#pragma unroll
                    for (int i = 0; i < 4; i++) v[8 + i] = (float)p[32 + 4 * c + i];
                } else {
#pragma unroll
                    for (int i = 0; i < DK / 32; i++) load8(p + (DK / 4) * c + 8 * i, a.q_vec, v + 8 * i);
                }
            }
            float top = 0.f, sum = 0.f;
            bool bad = false;
#pragma unroll
            for (int i = 0; i < DK / 4; i++) {
                top = fmaxf(top, fabsf(v[i]));
                bad |= !(fabsf(v[i]) <= FLT_MAX);
                sum += v[i];
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            bad |= __shfl_xor_sync(0xffffffffu, (int)bad, 1) != 0;
            bad |= __shfl_xor_sync(0xffffffffu, (int)bad, 2) != 0;
            // 2^e <= top < 2^(e+1) goes to 2^14: f16's largest values
            int e = (int)((__float_as_uint(top) >> 23) & 255) - 127;
            e = min(max(e, -100), 127);
            const float up = __uint_as_float((uint32_t)(14 - e + 127) << 23);
            float fac0 = a.scale_log2e * __uint_as_float((uint32_t)(e - 14 + 127) << 23) * 16777216.f;
            float fac1 = a.scale_log2e * sum;
            if (bad) fac0 = fac1 = __uint_as_float(0x7fc00000u);
            float q1 = 0.f, q2 = 0.f;  // sums of the fixed-point terms: exact
            auto put = [&](int k, int half, float x0, float x1) {  // operand `half` of k-step k
                const float mul = half ? 0.0625f : 1.f;  // the second operand's codes come 16-fold
                uint32_t hi, lo = 0;
                if (QS == 2) {
                    // multiples of 16 up to 2^15, then of 2^-8 up to 8
                    const float a0 = __fmul_rn(rintf(x0 * 0.0625f), 16.f), a1 = __fmul_rn(rintf(x1 * 0.0625f), 16.f);
                    const float b0 = __fmul_rn(rintf((x0 - a0) * 256.f), 0.00390625f), b1 = __fmul_rn(rintf((x1 - a1) * 256.f), 0.00390625f);
                    q1 += a0 + a1, q2 += b0 + b1;
                    hi = pack_half2(a0 * mul, a1 * mul), lo = pack_half2(b0 * mul, b1 * mul);
                } else {
                    hi = pack_half2(x0 * mul, x1 * mul);
                }
                const int at = (t * KS + k) * 2 * QS + half * QS;
                if constexpr (Sh::Q_SMEM) {
                    qsm[at * 32] = hi;
                    if (QS == 2) qsm[(at + 1) * 32] = lo;
                } else {
                    qreg[at] = hi;
                    if (QS == 2) qreg[at + QS - 1] = lo;
                }
            };
#pragma unroll
            for (int i = 0; i < DK / 4; i++) v[i] = bad ? 0.f : v[i] * up;
#pragma unroll
            for (int w = 0; w < DK / 32; w++) {
                const float* y = v + 8 * w;
                put(2 * w, 0, y[0], y[4]);
                put(2 * w, 1, y[1], y[5]);
                put(2 * w + 1, 0, y[2], y[6]);
                put(2 * w + 1, 1, y[3], y[7]);
            }
            if constexpr (DK == 48) {
                put(2, 0, v[8], v[10]);
                put(2, 1, v[9], v[11]);
            }
            if (QS == 2) {
                q1 += __shfl_xor_sync(0xffffffffu, q1, 1);
                q2 += __shfl_xor_sync(0xffffffffu, q2, 1);
                q1 += __shfl_xor_sync(0xffffffffu, q1, 2);
                q2 += __shfl_xor_sync(0xffffffffu, q2, 2);
            }
            const int hi = on ? (int)min(max(rows.pos0 + x / a.group, -1LL), 0x7fffffffLL) : -1;
#pragma unroll
            for (int j = 0; j < 2; j++) {
                f0[t][j] = __shfl_sync(0xffffffffu, fac0, 4 * (2 * c + j));
                f1[t][j] = __shfl_sync(0xffffffffu, fac1, 4 * (2 * c + j));
                seen_hi[t][j] = __shfl_sync(0xffffffffu, hi, 4 * (2 * c + j));
                if (QS == 2) {  // -8 of the codes' unit, 2^-24
                    mid[t][j][0] = __shfl_sync(0xffffffffu, q1, 4 * (2 * c + j)) * -4.76837158203125e-7f;
                    mid[t][j][1] = __shfl_sync(0xffffffffu, q2, 4 * (2 * c + j)) * -4.76837158203125e-7f;
                }
            }
        }
        // tiles wholly inside every row's span need no masks
        const int x_last = min((b + 1) * 8 * NT, nrows) - 1;
        const long long p_first = rows.pos0 + (b * 8 * NT) / a.group, p_last = rows.pos0 + x_last / a.group;

        float acc[NT][MT][4], M[NT][2], l[NT][2], mn[NT][2];
#pragma unroll
        for (int t = 0; t < NT; t++) {
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[t][i][j] = 0.f;
#pragma unroll
            for (int j = 0; j < 2; j++) M[t][j] = -INFINITY, l[t][j] = mn[t][j] = 0.f;
        }

        for (int i = 0; i < m; i++) {
            asm volatile("cp.async.wait_group %0;\n" ::"n"(ATT_STAGES - 2) : "memory");
            __syncwarp();
            const int st = i % ATT_STAGES;
            const bool page_ok = (okbits >> st) & 1;
            issue();  // into the stage read in the last round
            const uint8_t* tile = ring + st * TB;
            const int k0 = tl.at(off + i) * KV4_TILE;

            // scores: keys g and g + 8 against query rows 2 c, 2 c + 1
            float sc[NT][4], sc2[QS == 2 ? NT : 1][4];
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    sc[t][j] = QS == 2 ? mid[QS == 2 ? t : 0][j & 1][0] : 0.f;
                    if (QS == 2) sc2[QS == 2 ? t : 0][j] = mid[QS == 2 ? t : 0][j & 1][1];
                }
            auto qop = [&](int t, int k, int half, int term) -> uint32_t {
                const int at = (t * KS + k) * 2 * QS + half * QS + term;
                if constexpr (Sh::Q_SMEM) return qsm[at * 32];
                else return qreg[at];
            };
            auto step = [&](int k, uint32_t x0, uint32_t x1, uint32_t y0, uint32_t y1) {
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    mma16816(sc[t], x0, y0, x1, y1, qop(t, k, 0, 0), qop(t, k, 1, 0));
                    if (QS == 2) mma16816(sc2[QS == 2 ? t : 0], x0, y0, x1, y1, qop(t, k, 0, QS - 1), qop(t, k, 1, QS - 1));
                }
            };
            const uint8_t *ka = tile + g * (DK / 2), *kb = tile + (g + 8) * (DK / 2);
            uint32_t wa[DK / 32], wb[DK / 32];
            if constexpr (DK == 128) {
                const uint4 x = *(const uint4*)(ka + 16 * c), y = *(const uint4*)(kb + 16 * c);
                wa[0] = x.x, wa[1] = x.y, wa[2] = x.z, wa[3] = x.w;
                wb[0] = y.x, wb[1] = y.y, wb[2] = y.z, wb[3] = y.w;
            } else if constexpr (DK == 64) {
                const uint2 x = *(const uint2*)(ka + 8 * c), y = *(const uint2*)(kb + 8 * c);
                wa[0] = x.x, wa[1] = x.y;
                wb[0] = y.x, wb[1] = y.y;
            } else {
                wa[0] = *(const uint32_t*)(ka + 4 * c);
                wb[0] = *(const uint32_t*)(kb + 4 * c);
            }
#pragma unroll
            for (int w = 0; w < DK / 32; w++) {
                step(2 * w, wa[w] & 0x000f000fu, wa[w] & 0x00f000f0u, wb[w] & 0x000f000fu, wb[w] & 0x00f000f0u);
                const uint32_t xa = wa[w] >> 8, xb = wb[w] >> 8;
                step(2 * w + 1, xa & 0x000f000fu, xa & 0x00f000f0u, xb & 0x000f000fu, xb & 0x00f000f0u);
            }
            if constexpr (DK == 48) {  // dimensions 32 .. 47: four codes a lane
                const uint32_t ha = *(const uint16_t*)(ka + 16 + 2 * c), hb = *(const uint16_t*)(kb + 16 + 2 * c);
                const uint32_t xa = __byte_perm(ha, 0, 0x4140), xb = __byte_perm(hb, 0, 0x4140);
                step(2, xa & 0x000f000fu, xa & 0x00f000f0u, xb & 0x000f000fu, xb & 0x00f000f0u);
            }
            const uint8_t* par = tile + 8 * (DK + DV);
            float2 kpa = unpack_half2(*(const uint32_t*)(par + 4 * g)), kpb = unpack_half2(*(const uint32_t*)(par + 4 * (g + 8)));
            float2 vpa = unpack_half2(*(const uint32_t*)(par + 64 + 4 * g)), vpb = unpack_half2(*(const uint32_t*)(par + 64 + 4 * (g + 8)));
            if (QS == 2) {  // the middle of the codes instead of the minimum
                kpa.y = __fmaf_rn(8.f, kpa.x, kpa.y), kpb.y = __fmaf_rn(8.f, kpb.x, kpb.y);
                vpa.y = __fmaf_rn(8.f, vpa.x, vpa.y), vpb.y = __fmaf_rn(8.f, vpb.x, vpb.y);
            }
            const float la = lg2(fmaxf(vpa.x, 5.9604645e-8f)), lb = lg2(fmaxf(vpb.x, 5.9604645e-8f));
            const bool whole = page_ok && k0 + 15 <= p_first && (a.window <= 0 || k0 > p_last - a.window || k0 + 15 < a.sink);
            uint32_t vis = 0xffffffffu;
            bool raise = false;
#pragma unroll
            for (int t = 0; t < NT; t++) {
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    if (QS == 2) sc[t][j] += sc2[QS == 2 ? t : 0][j], sc[t][2 + j] += sc2[QS == 2 ? t : 0][2 + j];
                    sc[t][j] = __fmaf_rn(kpa.x, sc[t][j] * f0[t][j], kpa.y * f1[t][j]);
                    sc[t][2 + j] = __fmaf_rn(kpb.x, sc[t][2 + j] * f0[t][j], kpb.y * f1[t][j]);
                }
                if (!whole) {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int key = k0 + g + (j >= 2 ? 8 : 0), hi = seen_hi[t][j & 1];
                        const bool ok = page_ok && key <= hi && (a.window <= 0 || key > hi - a.window || key < a.sink);
                        if (!ok) vis &= ~(1u << (4 * t + j));
                    }
                }
#pragma unroll
                for (int j = 0; j < 4; j++) raise |= ((vis >> (4 * t + j)) & 1) && sc[t][j] + (j >= 2 ? lb : la) > M[t][j & 1] + 4.f;
            }
            if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        float mx = M[t][j];
                        if ((vis >> (4 * t + j)) & 1) mx = fmaxf(mx, sc[t][j] + la);
                        if ((vis >> (4 * t + 2 + j)) & 1) mx = fmaxf(mx, sc[t][2 + j] + lb);
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                        const float r = mx == -INFINITY ? 1.f : ex2(M[t][j] - mx);
                        M[t][j] = mx;
                        l[t][j] *= r;
                        mn[t][j] *= r;
#pragma unroll
                        for (int k = 0; k < MT; k++) acc[t][k][j] *= r, acc[t][k][2 + j] *= r;
                    }
            }
            // weights, and their operands: rows of the transpose are query rows
            uint32_t wop[NT][2][WS];
#pragma unroll
            for (int t = 0; t < NT; t++) {
                float w[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const bool ok = (vis >> (4 * t + j)) & 1;
                    const float p = ok ? ex2(sc[t][j] - M[t][j & 1]) : 0.f;
                    const float2 vp = j >= 2 ? vpb : vpa;
                    w[j] = ok ? p * vp.x : 0.f;
                    l[t][j & 1] += p;
                    mn[t][j & 1] = __fmaf_rn(p, ok ? vp.y : 0.f, mn[t][j & 1]);
                }
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    const uint32_t hi = pack_half2(w[2 * half], w[2 * half + 1]);
                    wop[t][half][0] = transpose8(hi);
                    if (WS == 2) {
                        const float2 r = unpack_half2(hi);
                        wop[t][half][WS - 1] = transpose8(pack_half2(w[2 * half] - r.x, w[2 * half + 1] - r.y));
                    }
                }
            }
            // values: lane (g, c) holds dimensions 8 (VW g + w) .. + 7 of keys 2c, 2c+1, 2c+8, 2c+9
            const uint8_t* vt = tile + 8 * DK + g * 4 * VW;
            uint32_t vw[4][VW];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint8_t* p = vt + (2 * c + (j & 1) + (j >= 2 ? 8 : 0)) * (DV / 2);
                if constexpr (VW == 2) {
                    const uint2 x = *(const uint2*)p;
                    vw[j][0] = x.x, vw[j][1] = x.y;
                } else {
                    vw[j][0] = *(const uint32_t*)p;
                }
            }
#pragma unroll
            for (int w = 0; w < VW; w++)
#pragma unroll
                for (int quarter = 0; quarter < 4; quarter++) {
                    // dimensions 2 quarter (row g), 2 quarter + 1 (row g + 8)
                    const uint32_t sel = quarter < 2 ? 0x5410 : 0x7632;
                    const uint32_t x = __byte_perm(vw[0][w], vw[1][w], sel) >> (quarter & 1 ? 8 : 0);
                    const uint32_t y = __byte_perm(vw[2][w], vw[3][w], sel) >> (quarter & 1 ? 8 : 0);
                    uint32_t a0 = x & 0x000f000fu, a1 = x & 0x00f000f0u, a2 = y & 0x000f000fu, a3 = y & 0x00f000f0u;
                    if (MID) a0 = code_mid(a0), a1 = code16_mid(a1), a2 = code_mid(a2), a3 = code16_mid(a3);
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        float* d = acc[t][4 * w + quarter];
                        if constexpr (MID) {
                            float z[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                            for (int term = 0; term < WS; term++) mma16816(z, a0, a1, a2, a3, wop[t][0][term], wop[t][1][term]);
#pragma unroll
                            for (int j = 0; j < 4; j++) d[j] += z[j];
                        } else {
#pragma unroll
                            for (int term = 0; term < WS; term++) mma16816(d, a0, a1, a2, a3, wop[t][0][term], wop[t][1][term]);
                        }
                    }
                }
        }
        asm volatile("cp.async.wait_group 0;\n" ::: "memory");

        // this run's part of the unit: sums over the keys' lanes, 2^24 back
        const bool starts = off == 0, ends = off + m == tl.n;
        float* part = a.parts + ((size_t)wid * 2 + (starts ? 1 : 0)) * Sh::PART;
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
#pragma unroll
                for (int o = 4; o < 32; o *= 2) {
                    l[t][j] += __shfl_xor_sync(0xffffffffu, l[t][j], o);
                    mn[t][j] += __shfl_xor_sync(0xffffffffu, mn[t][j], o);
                }
                const int y = 8 * t + 2 * c + j, x = b * 8 * NT + y;  // query row in the block, in the sequence
                const float norm = starts && ends ? (l[t][j] == 0.f ? 0.f : 1.f / l[t][j]) : 1.f;
                T* o = out + (rows.first + x / a.group) * a.o_row + (h * a.group + x % a.group) * a.o_head;
#pragma unroll
                for (int w = 0; w < VW; w++) {
                    float v[8];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        v[2 * k] = __fmaf_rn(acc[t][4 * w + k][j], MID ? 1.f : 16777216.f, mn[t][j]) * norm;
                        v[2 * k + 1] = __fmaf_rn(acc[t][4 * w + k][2 + j], MID ? 1.f : 1048576.f, mn[t][j]) * norm;
                    }
                    const int d0 = 8 * (VW * g + w);
                    if (starts && ends) {
                        if (x < nrows) store8(o + d0, a.o_vec, v);
                    } else {
                        store8(part + y * DV + d0, true, v);
                    }
                }
                if (!(starts && ends) && g == 0) {
                    part[8 * NT * DV + y] = M[t][j];
                    part[8 * NT * (DV + 1) + y] = l[t][j];
                }
            }
        if (starts && !ends && lane == 0) {
            const int further = (int)((cur + tl.n - 1) / share - wid);
            a.joins[wid] = make_int4(s, h, b, further);
        }

        // the next unit
        cur += m;
        if (cur >= end) break;
        off = 0;
        if (++b * 8 * NT >= nrows) {
            b = 0;
            if (++h == H) {
                h = 0;
                do rows = seq_rows(a, ++s);
                while (rows.n == 0);
            }
        }
        tl = block_tiles<NT>(a, rows, b);
    }
}

// out = sum_w 2^(M_w - M) acc_w / sum_w 2^(M_w - M) l_w over the warps w that
// share a unit, in their order. A CTA per warp of the first kernel; those
// where no cut unit starts return at once.
template <int DV, int NT, typename T>
__global__ void __launch_bounds__(128) kv4_join_kernel(AttendArgs a, T* __restrict__ out) {
    constexpr int PART = 8 * NT * (DV + 2), ROWS = 128 / DV;
    const int4 job = a.joins[blockIdx.x];
    if (job.w < 0) return;
    const SeqRows rows = seq_rows(a, job.x);
    const int y = blockIdx.y * ROWS + threadIdx.x / DV, d = threadIdx.x % DV, x = job.z * 8 * NT + y;
    if (x >= rows.n * a.group) return;
    auto part = [&](int i) { return a.parts + ((size_t)(blockIdx.x + i) * 2 + (i == 0)) * PART; };
    float M = -INFINITY;
    for (int i = 0; i <= job.w; i++) M = fmaxf(M, __ldg(part(i) + 8 * NT * DV + y));
    float l = 0.f, v = 0.f;
    for (int i = 0; i <= job.w; i++) {
        const float* p = part(i);
        const float m = __ldg(p + 8 * NT * DV + y);
        const float li = __ldg(p + 8 * NT * (DV + 1) + y);
        const float r = m == M ? 1.f : ex2(m - M);
        l = __fmaf_rn(li, r, l);
        v = __fmaf_rn(__ldg(p + y * DV + d), r, v);
    }
    v = l == 0.f ? 0.f : v / l;
    T* o = out + (rows.first + x / a.group) * a.o_row + (job.y * a.group + x % a.group) * a.o_head;
    o[d] = (T)v;
}

// Query rows a block: the fewest blocks of 8, 16 or 32 rows that hold what a
// sequence brings on average.
static int query_tiles(const nd_kv4* kv, int group) {
    const long long mean = ((long long)kv->rows + kv->seqs - 1) / kv->seqs * group;
    return mean <= 8 ? 1 : mean <= 16 ? 2 : 4;
}

static int attend_ctas(int nt) { return device_sm_count() * (nt == 1 ? 4 : nt == 2 ? 3 : 2); }

static size_t attend_ws_bytes(int nt, int dv, int ctas) {
    const size_t warps = (size_t)ctas * ATT_WARPS;
    return warps * (sizeof(int4) + 2 * sizeof(float) * 8 * nt * (dv + 2));
}

template <int DK, int DV, int NT, typename T>
static void attend_launch(const AttendArgs& a0, const void* q, void* out, void* ws, int ctas, cudaStream_t st) {
    using Sh = AttendShape<DK, DV, NT, T>;
    AttendArgs a = a0;
    a.joins = (int4*)ws;
    a.parts = (float*)((char*)ws + (size_t)ctas * ATT_WARPS * sizeof(int4));
    auto kernel = kv4_attend_kernel<DK, DV, NT, T>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::SMEM);
    if (e != cudaSuccess) throw std::runtime_error(std::string("nd_op_kv4_attend: ") + cudaGetErrorString(e));
    kernel<<<ctas, 32 * ATT_WARPS, Sh::SMEM, st>>>(a, (const T*)q, (T*)out);
    op_launched("nd_op_kv4_attend");
    kv4_join_kernel<DV, NT, T><<<dim3(ctas * ATT_WARPS, 8 * NT * DV / 128), 128, 0, st>>>(a, (T*)out);
    op_launched("nd_op_kv4_attend");
}

template <int DK, int DV, typename T>
static void attend_nt(int nt, const AttendArgs& a, const void* q, void* out, void* ws, int ctas, cudaStream_t st) {
    if (nt == 1) attend_launch<DK, DV, 1, T>(a, q, out, ws, ctas, st);
    else if (nt == 2) attend_launch<DK, DV, 2, T>(a, q, out, ws, ctas, st);
    else attend_launch<DK, DV, 4, T>(a, q, out, ws, ctas, st);
}

template <int DK, int DV>
static void attend_type(int type, int nt, const AttendArgs& a, const void* q, void* out, void* ws, int ctas, cudaStream_t st) {
    if (type == ND_F32) attend_nt<DK, DV, float>(nt, a, q, out, ws, ctas, st);
    else if (type == ND_F16) attend_nt<DK, DV, __half>(nt, a, q, out, ws, ctas, st);
    else attend_nt<DK, DV, __nv_bfloat16>(nt, a, q, out, ws, ctas, st);
}

}  // namespace nd

using namespace nd;

extern "C" {

unsigned long long nd_op_kv4_attend_ws(const nd_kv4* kv, int q_heads) {
    unsigned long long bytes = 0;
    op_call([&] {
        kv4_args(kv, "nd_op_kv4_attend_ws");
        if (q_heads < 1 || q_heads % kv->heads) throw std::runtime_error("nd_op_kv4_attend_ws: q_heads must be a multiple of heads");
        OnDevice on(kv->device, "nd_op_kv4_attend_ws");
        const int nt = query_tiles(kv, q_heads / kv->heads);
        bytes = attend_ws_bytes(nt, kv->dv, attend_ctas(nt));
    });
    return bytes;
}

int nd_op_kv4_attend(const nd_kv4* kv, int type, const void* q, long long q_row, long long q_head, int q_heads, float scale,
                     int window, int sink, void* out, long long o_row, long long o_head, void* ws, unsigned long long ws_bytes,
                     void* stream) {
    return op_call([&] {
        const char* what = "nd_op_kv4_attend";
        auto fail = [&](const std::string& m) { throw std::runtime_error(std::string(what) + ": " + m); };
        AttendArgs a{};
        a.kv = kv4_args(kv, what);
        if (a.kv.rows == 0) return;
        if (q_heads < 1 || q_heads % a.kv.heads) fail("q_heads must be a multiple of heads");
        a.group = q_heads / a.kv.heads;
        if (a.group > 64) fail("more than 64 query heads a kv head");
        if ((long long)a.kv.rows * a.group > 0x7fffffffLL / 2) fail("too many rows");
        if (window < 0 || sink < 0) fail("window and sink must not be negative");
        if (!(fabsf(scale) <= FLT_MAX)) fail("scale must be finite");
        kv4_check_rows(what, type, q, q_row, q_head);
        kv4_check_out(what, type, out, o_row, o_head, a.kv.rows, q_heads, kv->dv);
        if (!ws || (uintptr_t)ws % 16) fail("the workspace must be 16-byte aligned");
        a.q_row = q_row, a.q_head = q_head, a.o_row = o_row, a.o_head = o_head;
        a.window = window, a.sink = sink;
        a.scale_log2e = (float)((double)scale * 1.4426950408889634);
        a.q_vec = kv4_vec(type, q, q_row, q_head), a.o_vec = kv4_vec(type, out, o_row, o_head);
        OnDevice on(kv->device, what);
        const int nt = query_tiles(kv, a.group), ctas = attend_ctas(nt);
        if (ws_bytes < attend_ws_bytes(nt, kv->dv, ctas)) fail("the workspace is too small");
        cudaStream_t st = (cudaStream_t)stream;
        if (kv->dk == 48) attend_type<48, 64>(type, nt, a, q, out, ws, ctas, st);
        else if (kv->dk == 64) attend_type<64, 64>(type, nt, a, q, out, ws, ctas, st);
        else attend_type<128, 128>(type, nt, a, q, out, ws, ctas, st);
    });
}

}  // extern "C"
