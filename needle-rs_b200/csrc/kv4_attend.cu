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
// Weights p sv are split into two f16 terms (22 bits, down to 2^-36 of the
// row's largest weight, see ATT_TOP) for f32 and f16 rows; bf16 rows take
// one: its 2^-12 is far below the output's own 2^-9.
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
// - sums of 16 rounds are carried in f64 (ATT_ROUNDS).
// Measured: 6e-7 of the result against 64 bits where the plain way had 4e-5
// (keys and values with outlying channels); below 2e-6 over a run of 32,768
// equal keys behind one that is 10 to 18 nats ahead.
//
// A warp keeps the softmax's running reference M per query row (a power-of-
// two argument: scores carry log2 e) and rescales only when a new exponent
// passes it by more than 4, since only the quotient counts. The reference is
// taken over score + log2 sv, so that the f16 weight p sv is at most 2^15
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
#include "kv4_attend.cuh"
#include "kv4_host.h"
#include "tc.cuh"

namespace nd {

constexpr int ATT_WARPS = 4;
constexpr int ATT_KT = 2, ATT_STAGES = 3;
// Rounds after which a run's sums go to memory (f64 for f32 rows) and begin
// anew: in f32 small terms beside a large sum lose up to 2^-24 of it each,
// which thousands of equal ones add up. Few runs are that long.
__host__ __device__ constexpr int ATT_ROUNDS(bool f32) { return f32 ? 16 : 32; }
constexpr int ATT_CTAS(int nt, int dv) { return nt == 2 || dv == 128 ? 3 : 4; }  // an SM: what registers and shared memory allow
// Tiles: a shorter run of a cut unit costs more to join than it takes.
constexpr int ATT_MIN_SHARE = 8;
// What beginning and ending a unit costs a warp, in tiles: without it a warp
// that meets many short units is the last by far (8 sequences, one of a
// single position among lengths up to 32768: 70 us instead of 57, before sums
// were carried on).
constexpr int ATT_UNIT_COST = 4;
// 16-bit rows that would be cut go to the tcgen05 kernel from this many query
// rows a sequence and kv head on average, and this many tiles by blocks of
// eight rows: it takes 30 us (heads of 128: 40) at the least. Measured (us,
// this kernel, that one; bf16): 4 heads of 128 a kv head, 4 sequences of 64 rows
// over 740 positions 24, 40; 8 of them 40, 43; 16 of them 61, 56; one of 128
// over 2000 45, 42, over 4000 65, 50; 6 heads of 64, one of 512 over 740 47, 34,
// of 128 over 4096 33, 34, over 20000 66, 54.
constexpr int ATT_TC_ROWS = 128;
constexpr long long ATT_TC_WORK(int dv) { return dv == 128 ? 1 << 16 : 1 << 15; }
// Calls whose units all have few tiles take them whole, a warp or, where units
// are too few to fill the GPU twice, a CTA a unit, and need no second kernel
// and no place in a list, 8 us of the cut units' time. A warp a unit: up to
// ATT_WARP_TILES, and where there are more units than CTAs at once to
// ATT_WARP_MOST (a warp's own time shows with more).
// A CTA: up to ATT_CTA_TILES, half for two rounds. Measured (us; one token of 6
// heads a kv head, f32; cut units, a warp, a CTA a unit): 32 sequences of up to
// 256 positions 14.4, 10.1, 6.7; 512 of them 21.9, 14.7, 16.1; 32 of up to 1000
// 14.9, -, 11.1; 512 of up to 640 29.0, 27.8, 23.4; 1024 of up to 400 35.5,
// 25.9, 34.4; of up to 740 49.6, 43.4, -; of up to 1000 59.0, 56.0, 57.5, and
// in a window of 74 tiles, five tokens, 256 sequences 51.5, 54.1. Heads of 128
// bf16, 256 of up to 400 39.0, 34.8, 47.2; 128 of up to 740 34.0, 37.5, -. Whole
// prompts of 118 rows, 6 heads, bf16, 256 of them: a warp a unit 79, on tcgen05 134.
// Tiles here are what the table's columns or the window could hold, as the
// host knows no lengths: with columns for 4096 positions the same calls are cut
// or go to tcgen05 (one session 4.8, 10.3; 1024 sequences of up to 256 19.1, 31.2;
// 32 of them 6.2, 15.4; 16 prompts of 118 rows 10.5, 32.3).
constexpr int ATT_WARP_TILES = 16, ATT_CTA_TILES = 128;
constexpr int ATT_WARP_MOST(int dv) { return dv == 128 ? 32 : 48; }
static_assert(ATT_WARP_MOST(64) <= ATT_ROUNDS(false) * ATT_KT && ATT_CTA_TILES / ATT_WARPS + ATT_KT <= ATT_ROUNDS(false) * ATT_KT, "whole units are not LONG");

// Whole units are numbered without sums. Places 0 .. seqs - 1 are the
// sequences' first blocks; the further blocks of sequence s are at most the
// places from further_place(s) to further_place(s + 1): ceil(y - x) - 1 <=
// floor(y) - floor(x). Places that no block has are left at once.
template <int NT>
__device__ __forceinline__ int further_place(const AttendArgs& a, int s) {
    return (int)((long long)kv4_first_row(a.kv, s) * a.group.d / (8 * NT));
}

// The sequence of place u (by the whole warp, 32 sequences at a time) and its block.
template <int NT>
__device__ __forceinline__ int seq_of_place(const AttendArgs& a, int u, int lane, int* block) {
    *block = 0;
    if (u < a.kv.seqs) return u;
    u -= a.kv.seqs;
    int lo = 0, size = a.kv.seqs;  // how many begin at or before u
    while (size > 0) {
        const int step = (size + 31) / 32, at = lane * step + step - 1;
        const bool before = at < size && further_place<NT>(a, lo + at) <= u;
        const int c = __popc(__ballot_sync(0xffffffffu, before));
        lo += c * step;
        size = min(step - 1, size - c * step);
    }
    if (lo > 0) *block = 1 + u - further_place<NT>(a, lo - 1);
    return *block > 0 ? lo - 1 : -1;  // no place before its first, should `start` not ascend
}

// What a sequence and kv head adds to the list of work: each unit its cost
// and then its tiles.
template <int NT>
__device__ __forceinline__ long long seq_work(const AttendArgs& a, const SeqRows& r) {
    const int blocks = (r.n * (int)a.group.d + 8 * NT - 1) / (8 * NT);
    long long t = 0;
    for (int b = 0; b < blocks; b++) t += block_tiles<NT>(a, r, b).n + ATT_UNIT_COST;
    return t;
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
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, uint32_t bytes) {  // 16 of them, or none and zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

template <int DK, int DV, int NT, typename T>
struct AttendShape {
    static constexpr int TB = kv4_tile_bytes(DK, DV);
    static constexpr bool F32 = std::is_same<T, float>::value;
    static constexpr int QS = F32 ? 2 : 1;                                     // f16 terms of a query value
    static constexpr int WS = std::is_same<T, __nv_bfloat16>::value ? 1 : 2;  // f16 terms of a weight
    static constexpr int KSTEPS = DK / 16;
    static constexpr int QOPS = NT * KSTEPS * QS;  // a query block's operands: pairs of registers
    static constexpr bool Q_SMEM = QOPS > 16;      // else they stay in registers
    // Tiles a round of the main loop, and rounds in flight: two tiles give a
    // warp two independent chains of products, and share a round's overhead.
    static constexpr int KT = ATT_KT, STAGES = ATT_STAGES;
    // For one block of eight rows the warps of a CTA join their parts in
    // shared memory first: decoding cuts few units into many parts.
    static constexpr bool MERGE = NT == 1;
    static constexpr int PART = 8 * NT * (DV + 2);  // floats
    static constexpr int SLOTS = STAGES * KT * TB;
    static constexpr int RING = SLOTS > 4 * PART || !MERGE ? SLOTS : 4 * PART;
    static constexpr int QBYTES = Q_SMEM ? QOPS * 256 : 0;
    static constexpr int WARP_SMEM = RING + QBYTES + (MERGE ? 4 * PART : 0);
    static constexpr int SMEM = ATT_WARPS * WARP_SMEM, WHOLE_SMEM = ATT_WARPS * (RING + QBYTES);
    static constexpr int CTAS = ATT_CTAS(NT, DV);
};

// A part of 8 rows as a warp holds it.
template <int DV>
struct PartRegs {
    float v[2][DV / 8], M[2], l[2];  // rows 2 c, 2 c + 1; dimensions (DV / 8) g ..
    __device__ __forceinline__ void load(const float* p, int g, int c) {
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const int y = 2 * c + j;
#pragma unroll
            for (int k = 0; k < DV / 32; k++) *(float4*)&v[j][4 * k] = *(const float4*)(p + y * DV + (DV / 8) * g + 4 * k);
            M[j] = p[8 * DV + y];
            l[j] = p[8 * (DV + 1) + y];
        }
    }
    // the quotients, for rows x0 ..
    template <typename T>
    __device__ __forceinline__ void write(const OutRows<T>& to, int x0, int g, int c) {
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const int x = x0 + 2 * c + j;
            const float norm = l[j] == 0.f ? 0.f : 1.f / l[j];
#pragma unroll
            for (int k = 0; k < DV / 8; k++) v[j][k] *= norm;
            if (x < to.nrows)
#pragma unroll
                for (int k = 0; k < DV / 64; k++) store8(to.at(x) + (DV / 8) * g + 8 * k, to.a.o_vec, v[j] + 8 * k);
        }
    }
    __device__ __forceinline__ void add(const PartRegs& o) {
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const float m = fmaxf(M[j], o.M[j]);
            const float r = ex2(M[j] - m), s = ex2(o.M[j] - m);
            M[j] = m;
            l[j] = __fmaf_rn(l[j], r, o.l[j] * s);
#pragma unroll
            for (int k = 0; k < DV / 8; k++) v[j][k] = __fmaf_rn(v[j][k], r, o.v[j][k] * s);
        }
    }
};


// A warp's part of a unit: tiles off .. off + m - 1 of query block b of
// sequence s and kv head h. With `part` NULL they are all it has and the
// result goes to its place; else the sums go to `part`, unnormalised. LONG:
// it may have more rounds than sums in f32 should (ATT_ROUNDS).
template <int DK, int DV, int NT, typename T, bool LONG>
__device__ __forceinline__ void attend_part(const AttendArgs& a, const T* __restrict__ q, T* __restrict__ out, int s, int h, int b,
                                            const SeqRows& rows, const Tiles& tl, int off, int m, uint8_t* ring, uint2* qsm0,
                                            float* part) {
    using Sh = AttendShape<DK, DV, NT, T>;
    constexpr int TB = Sh::TB, QS = Sh::QS, WS = Sh::WS, KS = Sh::KSTEPS, MT = DV / 16, VW = DV / 64, KT = Sh::KT, STAGES = Sh::STAGES;
    constexpr bool F32 = Sh::F32;
    constexpr int ROUNDS = ATT_ROUNDS(F32);
    const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int nrows = rows.n * (int)a.group.d;
    const uint32_t ring_s = (uint32_t)__cvta_generic_to_shared(ring) + lane * 16;
    uint2* qsm = qsm0 + lane;

    // addresses of the next tiles, 32 at a time, one batch ahead; 0: no such page
    const int32_t* trow = a.kv.table + (size_t)s * a.kv.table_stride;
    const uint8_t* head = a.kv.pool + (size_t)h * a.kv.page_tiles * TB;
    auto fetch = [&](int i) -> unsigned long long {
        if (i >= off + m) return 0;
        const int t = tl.at(i), p = a.page_tiles(t);
        const int page = p < a.kv.max_pages ? __ldg(trow + p) : -1;
        if (page < 0 || page >= a.kv.num_pages) return 0;
        return (unsigned long long)(head + (size_t)page * a.kv.page_stride + (size_t)(t - p * a.kv.page_tiles) * TB);
    };
    unsigned long long src = fetch(off + lane), src_next = fetch(off + 32 + lane);
    uint32_t have = 0;  // bit k: the tile issued k issues ago exists (others are zeros in the ring)
    int issued = 0;
    uint32_t put_at = 0;
    auto issue = [&]() {
#pragma unroll
        for (int u = 0; u < KT; u++) {
            const unsigned long long from = __shfl_sync(0xffffffffu, src, (issued + u) & 31);
            const uint32_t bytes = from ? 16 : 0;
            have = have << 1 | (from != 0);
            const uint8_t* p = (from ? (const uint8_t*)from : a.kv.pool) + lane * 16;
            const uint32_t d = ring_s + put_at + u * TB;
#pragma unroll
            for (int j = 0; j < TB / 512; j++) copy16(d + j * 512, p + j * 512, bytes);
            if (TB % 512 && lane * 16 < TB % 512) copy16(d + TB / 512 * 512, p + TB / 512 * 512, bytes);
        }
        put_at = put_at == (STAGES - 1) * KT * TB ? 0 : put_at + KT * TB;
        issued += KT;
        if (__builtin_expect((issued & 31) == 0, 0)) {
            src = src_next;
            src_next = fetch(off + issued + 32 + lane);
        }
        asm volatile("cp.async.commit_group;\n" ::: "memory");
    };
    __syncwarp();  // the ring's last tile has been read by every lane
#pragma unroll 1
    for (int i = 0; i < STAGES - 1; i++) issue();

    // the query block: lane (g, c) holds of query row 8 t + g the
    // dimensions whose codes it will hold of every key
    uint2 qreg[Sh::Q_SMEM ? 1 : Sh::QOPS];
    f32x2 f0[NT], f1[NT], mid[F32 ? NT : 1][2];
    int seen_hi[NT][2];
#pragma unroll
    for (int t = 0; t < NT; t++) {
        const int x = b * 8 * NT + 8 * t + g;
        const bool on = x < nrows;
        float v[DK / 4];
#pragma unroll
        for (int i = 0; i < DK / 4; i++) v[i] = 0.f;
        const int tok = a.group(x);
        if (on) {
            const T* p = q + (long long)(rows.first + tok) * a.q_row + (long long)(h * (int)a.group.d + x - tok * (int)a.group.d) * a.q_head;
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
        const int e = max((int)(__float_as_uint(top) >> 23) - 127, -100);
        const float up = bad ? 0.f : __uint_as_float((uint32_t)(14 - min(e, 127) + 127) << 23);
        float fac0 = a.scale_log2e * __uint_as_float((uint32_t)(min(e, 127) - 14 + 127) << 23) * 16777216.f;
        float fac1 = a.scale_log2e * sum;
        if (bad) fac0 = fac1 = __uint_as_float(0x7fc00000u);
        float q1 = 0.f, q2 = 0.f;  // sums of the fixed-point terms: exact
        auto terms = [&](float x0, float x1, float mul, uint32_t& hi, uint32_t& lo) {
            if (F32) {
                // multiples of 16 up to 2^15, then of 2^-8 up to 8
                const float a0 = rintf(x0 * 0.0625f) * 16.f, a1 = rintf(x1 * 0.0625f) * 16.f;
                const float b0 = rintf((x0 - a0) * 256.f) * 0.00390625f, b1 = rintf((x1 - a1) * 256.f) * 0.00390625f;
                q1 += a0 + a1, q2 += b0 + b1;
                hi = pack_half2(a0 * mul, a1 * mul), lo = pack_half2(b0 * mul, b1 * mul);
            } else {
                hi = pack_half2(x0 * mul, x1 * mul);
            }
        };
        // operands of k-step k: codes (x0, x1) as they are, (y0, y1) 16-fold
        auto put = [&](int k, float x0, float x1, float y0, float y1) {
            uint2 hi, lo;
            terms(x0, x1, 1.f, hi.x, lo.x);
            terms(y0, y1, 0.0625f, hi.y, lo.y);
            const int at = (t * KS + k) * QS;
            if constexpr (Sh::Q_SMEM) {
                qsm[at * 32] = hi;
                if (F32) qsm[(at + 1) * 32] = lo;
            } else {
                qreg[at] = hi;
                if (F32) qreg[at + QS - 1] = lo;
            }
        };
#pragma unroll
        for (int i = 0; i < DK / 4; i++) v[i] = bad ? 0.f : v[i] * up;
#pragma unroll
        for (int w = 0; w < DK / 32; w++) {
            const float* y = v + 8 * w;
            put(2 * w, y[0], y[4], y[1], y[5]);
            put(2 * w + 1, y[2], y[6], y[3], y[7]);
        }
        if constexpr (DK == 48) put(2, v[8], v[10], v[9], v[11]);
        const int hi = on ? (int)min(max(rows.pos0 + tok, -1LL), 0x7fffffffLL) : -1;
        auto cols = [&](float x) { return pair(__shfl_sync(0xffffffffu, x, 8 * c), __shfl_sync(0xffffffffu, x, 8 * c + 4)); };
        f0[t] = cols(fac0);
        f1[t] = cols(fac1);
        seen_hi[t][0] = __shfl_sync(0xffffffffu, hi, 8 * c);
        seen_hi[t][1] = __shfl_sync(0xffffffffu, hi, 8 * c + 4);
        if (F32) {  // -8 of the codes' unit, 2^-24
            q1 += __shfl_xor_sync(0xffffffffu, q1, 1);
            q2 += __shfl_xor_sync(0xffffffffu, q2, 1);
            q1 += __shfl_xor_sync(0xffffffffu, q1, 2);
            q2 += __shfl_xor_sync(0xffffffffu, q2, 2);
            mid[F32 ? t : 0][0] = cols(q1 * -4.76837158203125e-7f);
            mid[F32 ? t : 0][1] = cols(q2 * -4.76837158203125e-7f);
        }
    }
    // tiles wholly inside every row's span need no masks
    const int x_last = min((b + 1) * 8 * NT, nrows) - 1;
    const long long p_first = rows.pos0 + a.group(b * 8 * NT), p_last = rows.pos0 + a.group(x_last);
    const int all_hi = (int)min(max(p_first, -1LL), 0x7fffffffLL) - 15;              // whole: k0 <= all_hi and
    const int all_lo = a.window > 0 ? (int)min(max(p_last - a.window, -1LL), 0x7fffffffLL) : -1;  // k0 > all_lo or k0 + 15 < sink

    float acc[NT][MT][4];
    f32x2 nM[NT], l[NT], mn[NT];  // -M, sum p, sum p mv for columns 2 c, 2 c + 1 (the sums over this lane's keys)
    // the sums of earlier rounds; through a pointer the compiler cannot see
    // through, so that they stay out of the registers
    typedef typename std::conditional<F32, double, float>::type Sum;
    Sum earlier[NT * (4 * MT + 4)];
    Sum* past = earlier;
    asm volatile("" : "+l"(past) : : "memory");
    auto sums = [&](auto&& f) {  // f(i, value) of every sum; replaces it
#pragma unroll
        for (int t = 0; t < NT; t++) {
#pragma unroll
            for (int k = 0; k < MT; k++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[t][k][j] = f(t * (4 * MT + 4) + 4 * k + j, acc[t][k][j]);
            float2 x = unpair(l[t]), y = unpair(mn[t]);
            x.x = f(t * (4 * MT + 4) + 4 * MT, x.x), x.y = f(t * (4 * MT + 4) + 4 * MT + 1, x.y);
            y.x = f(t * (4 * MT + 4) + 4 * MT + 2, y.x), y.y = f(t * (4 * MT + 4) + 4 * MT + 3, y.y);
            l[t] = pair(x.x, x.y), mn[t] = pair(y.x, y.y);
        }
    };
#pragma unroll
    for (int t = 0; t < NT; t++) {
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) acc[t][i][j] = 0.f;
        nM[t] = pair(-ATT_LOW, -ATT_LOW);
        l[t] = mn[t] = 0;
    }

    int key0 = tl.at(off) * KV4_TILE;
    uint32_t get_at = 0;
#pragma unroll 1
    for (int i = 0; i < m; i += KT) {
        if (LONG && __builtin_expect(i > 0 && i % (ROUNDS * KT) == 0, 0)) {
            const bool first = i == ROUNDS * KT;
            sums([&](int k, float x) {
                past[k] = first ? (Sum)x : past[k] + (Sum)x;
                return 0.f;
            });
        }
        asm volatile("cp.async.wait_group %0;\n" ::"n"(STAGES - 2) : "memory");
        __syncwarp();
        const uint32_t here = have >> ((STAGES - 2) * KT);  // bit KT - 1 - u: tile u of this round
        issue();  // into the slots read in the last round
        const uint8_t* round = ring + get_at;
        get_at = get_at == (STAGES - 1) * KT * TB ? 0 : get_at + KT * TB;
        int k0[KT];
#pragma unroll
        for (int u = 0; u < KT; u++) {
            k0[u] = key0;
            key0 = off + i + u + 1 == tl.sink ? tl.lo * KV4_TILE : key0 + KV4_TILE;
        }
        bool whole = true;
#pragma unroll
        for (int u = 0; u < KT; u++) whole &= k0[u] <= all_hi && (k0[u] > all_lo || k0[u] + 15 < a.sink);
        whole &= (here & ((1u << KT) - 1)) == (1u << KT) - 1;

        // scores: keys g and g + 8 against query rows 2 c, 2 c + 1
        float sc[KT][NT][4], sc2[F32 ? KT : 1][F32 ? NT : 1][4];
#pragma unroll
        for (int u = 0; u < KT; u++)
#pragma unroll
            for (int t = 0; t < NT; t++) {
                if (F32) {
                    const float2 x = unpair(mid[F32 ? t : 0][0]), y = unpair(mid[F32 ? t : 0][1]);
                    sc[u][t][0] = sc[u][t][2] = x.x, sc[u][t][1] = sc[u][t][3] = x.y;
                    float* z = sc2[F32 ? u : 0][F32 ? t : 0];
                    z[0] = z[2] = y.x, z[1] = z[3] = y.y;
                } else {
                    sc[u][t][0] = sc[u][t][1] = sc[u][t][2] = sc[u][t][3] = 0.f;
                }
            }
        auto qop = [&](int t, int k, int term) -> uint2 {
            const int at = (t * KS + k) * QS + term;
            if constexpr (Sh::Q_SMEM) return qsm[at * 32];
            else return qreg[at];
        };
        uint32_t wa[KT][DK / 32], wb[KT][DK / 32];
        float2 kpa[KT], kpb[KT], vpa[KT], vpb[KT];
#pragma unroll
        for (int u = 0; u < KT; u++) {
            const uint8_t *ka = round + u * TB + g * (DK / 2), *kb = ka + 4 * DK;
            if constexpr (DK == 128) {
                const uint4 x = *(const uint4*)(ka + 16 * c), y = *(const uint4*)(kb + 16 * c);
                wa[u][0] = x.x, wa[u][1] = x.y, wa[u][2] = x.z, wa[u][3] = x.w;
                wb[u][0] = y.x, wb[u][1] = y.y, wb[u][2] = y.z, wb[u][3] = y.w;
            } else if constexpr (DK == 64) {
                const uint2 x = *(const uint2*)(ka + 8 * c), y = *(const uint2*)(kb + 8 * c);
                wa[u][0] = x.x, wa[u][1] = x.y;
                wb[u][0] = y.x, wb[u][1] = y.y;
            } else {
                wa[u][0] = *(const uint32_t*)(ka + 4 * c);
                wb[u][0] = *(const uint32_t*)(kb + 4 * c);
            }
            const uint8_t* par = round + u * TB + 8 * (DK + DV) + 4 * g;
            kpa[u] = unpack_half2(*(const uint32_t*)par), kpb[u] = unpack_half2(*(const uint32_t*)(par + 32));
            vpa[u] = unpack_half2(*(const uint32_t*)(par + 64)), vpb[u] = unpack_half2(*(const uint32_t*)(par + 96));
        }
#pragma unroll
        for (int k = 0; k < KS; k++) {
            uint32_t x0[KT], x1[KT], y0[KT], y1[KT];
#pragma unroll
            for (int u = 0; u < KT; u++) {
                uint32_t xa, xb;
                if (DK == 48 && k == 2) {  // dimensions 32 .. 47: four codes a lane
                    const uint8_t* p = round + u * TB + g * (DK / 2) + 16 + 2 * c;
                    xa = __byte_perm(*(const uint16_t*)p, 0, 0x4140), xb = __byte_perm(*(const uint16_t*)(p + 4 * DK), 0, 0x4140);
                } else {
                    xa = wa[u][k / 2 < DK / 32 ? k / 2 : 0], xb = wb[u][k / 2 < DK / 32 ? k / 2 : 0];
                    if (k & 1) xa >>= 8, xb >>= 8;
                }
                x0[u] = xa & 0x000f000fu, x1[u] = xa & 0x00f000f0u, y0[u] = xb & 0x000f000fu, y1[u] = xb & 0x00f000f0u;
            }
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const uint2 o = qop(t, k, 0);
#pragma unroll
                for (int u = 0; u < KT; u++) mma16816(sc[u][t], x0[u], y0[u], x1[u], y1[u], o.x, o.y);
                if (F32) {
                    const uint2 o2 = qop(t, k, QS - 1);
#pragma unroll
                    for (int u = 0; u < KT; u++) mma16816(sc2[F32 ? u : 0][F32 ? t : 0], x0[u], y0[u], x1[u], y1[u], o2.x, o2.y);
                }
            }
        }
        f32x2 sa[KT][NT], sb[KT][NT];  // keys g, g + 8
        float ta[KT], tb[KT];          // a score may pass M by this much before M is raised
#pragma unroll
        for (int u = 0; u < KT; u++) {
            if (F32) {  // the middle of the codes instead of the minimum
                kpa[u].y = __fmaf_rn(8.f, kpa[u].x, kpa[u].y), kpb[u].y = __fmaf_rn(8.f, kpb[u].x, kpb[u].y);
                vpa[u].y = __fmaf_rn(8.f, vpa[u].x, vpa[u].y), vpb[u].y = __fmaf_rn(8.f, vpb[u].x, vpb[u].y);
            }
            ta[u] = ATT_TOP + 4.f - lg2(fmaxf(vpa[u].x, 5.9604645e-8f)), tb[u] = ATT_TOP + 4.f - lg2(fmaxf(vpb[u].x, 5.9604645e-8f));
            const f32x2 ksa = pair(kpa[u].x, kpa[u].x), ksb = pair(kpb[u].x, kpb[u].x);
            const f32x2 kma = pair(kpa[u].y, kpa[u].y), kmb = pair(kpb[u].y, kpb[u].y);
#pragma unroll
            for (int t = 0; t < NT; t++) {
                f32x2 da = pair(sc[u][t][0], sc[u][t][1]), db = pair(sc[u][t][2], sc[u][t][3]);
                if (F32) {
                    const float* z = sc2[F32 ? u : 0][F32 ? t : 0];
                    da = add2(da, pair(z[0], z[1])), db = add2(db, pair(z[2], z[3]));
                }
                sa[u][t] = fma2(mul2(da, f0[t]), ksa, mul2(f1[t], kma));
                sb[u][t] = fma2(mul2(db, f0[t]), ksb, mul2(f1[t], kmb));
            }
        }
        if (__builtin_expect(!whole, 0)) {
#pragma unroll
            for (int u = 0; u < KT; u++) {
                const bool in = here >> (KT - 1 - u) & 1;
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    auto mask = [&](f32x2 x, int key) {
                        float2 f = unpair(x);
                        const bool sunk = key < a.sink;
                        if (!(in && key <= seen_hi[t][0] && (a.window <= 0 || sunk || key > seen_hi[t][0] - a.window))) f.x = -INFINITY;
                        if (!(in && key <= seen_hi[t][1] && (a.window <= 0 || sunk || key > seen_hi[t][1] - a.window))) f.y = -INFINITY;
                        return pair(f.x, f.y);
                    };
                    sa[u][t] = mask(sa[u][t], k0[u] + g);
                    sb[u][t] = mask(sb[u][t], k0[u] + g + 8);
                }
            }
        }
        bool raise = false;
        float2 xa[KT][NT], xb[KT][NT];  // exponents
#pragma unroll
        for (int u = 0; u < KT; u++)
#pragma unroll
            for (int t = 0; t < NT; t++) {
                xa[u][t] = unpair(add2(sa[u][t], nM[t])), xb[u][t] = unpair(add2(sb[u][t], nM[t]));
                raise |= xa[u][t].x > ta[u] || xa[u][t].y > ta[u] || xb[u][t].x > tb[u] || xb[u][t].y > tb[u];
            }
        if (__builtin_expect(__any_sync(0xffffffffu, raise), 0)) {
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const float2 old = unpair(nM[t]);
                float m0 = -old.x, m1 = -old.y;
#pragma unroll
                for (int u = 0; u < KT; u++) {
                    const float2 fa = unpair(sa[u][t]), fb = unpair(sb[u][t]);
                    m0 = fmaxf(m0, fmaxf(fa.x + (4.f - ta[u]), fb.x + (4.f - tb[u])));
                    m1 = fmaxf(m1, fmaxf(fa.y + (4.f - ta[u]), fb.y + (4.f - tb[u])));
                }
#pragma unroll
                for (int o = 4; o < 32; o *= 2) {
                    m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, o));
                    m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, o));
                }
                const float r0 = ex2(-old.x - m0), r1 = ex2(-old.y - m1);
                const f32x2 r = pair(r0, r1);
                nM[t] = pair(-m0, -m1);
                l[t] = mul2(l[t], r);
                mn[t] = mul2(mn[t], r);
#pragma unroll
                for (int k = 0; k < MT; k++) acc[t][k][0] *= r0, acc[t][k][1] *= r1, acc[t][k][2] *= r0, acc[t][k][3] *= r1;
                if (LONG && i >= ROUNDS * KT)
#pragma unroll 1
                    for (int k = 0; k < 4 * MT + 4; k += 2) {
                        Sum* o = past + t * (4 * MT + 4) + k;
                        o[0] *= r0, o[1] *= r1;
                    }
#pragma unroll
                for (int u = 0; u < KT; u++) xa[u][t] = unpair(add2(sa[u][t], nM[t])), xb[u][t] = unpair(add2(sb[u][t], nM[t]));
            }
        }
        // weights, and their operands: rows of the transpose are query rows
        uint32_t wop[KT][NT][2][WS];
        f32x2 l1[NT], mn1[NT];  // of these tiles
#pragma unroll
        for (int u = 0; u < KT; u++) {
            const f32x2 vsa = pair(vpa[u].x, vpa[u].x), vsb = pair(vpb[u].x, vpb[u].x), vma = pair(vpa[u].y, vpa[u].y), vmb = pair(vpb[u].y, vpb[u].y);
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const f32x2 pa = pair(ex2(xa[u][t].x), ex2(xa[u][t].y)), pb = pair(ex2(xb[u][t].x), ex2(xb[u][t].y));
                l1[t] = u ? add2(l1[t], add2(pa, pb)) : add2(pa, pb);
                f32x2 wa2 = mul2(pa, vsa), wb2 = mul2(pb, vsb), ma = mul2(pa, vma), mb = mul2(pb, vmb);
                if (__builtin_expect(!whole, 0)) {  // a masked place may hold NaN or infinity
                    auto clean = [](f32x2 x, float2 e) {
                        const float2 f = unpair(x);
                        return pair(e.x == -INFINITY ? 0.f : f.x, e.y == -INFINITY ? 0.f : f.y);
                    };
                    wa2 = clean(wa2, xa[u][t]), wb2 = clean(wb2, xb[u][t]), ma = clean(ma, xa[u][t]), mb = clean(mb, xb[u][t]);
                }
                mn1[t] = u ? add2(mn1[t], add2(ma, mb)) : add2(ma, mb);
                const float2 fa = unpair(wa2), fb = unpair(wb2);
                const uint32_t ha = pack_half2(fa.x, fa.y), hb = pack_half2(fb.x, fb.y);
                wop[u][t][0][0] = transpose8(ha), wop[u][t][1][0] = transpose8(hb);
                if (WS == 2) {
                    const float2 ra = unpack_half2(ha), rb = unpack_half2(hb);
                    wop[u][t][0][WS - 1] = transpose8(pack_half2(fa.x - ra.x, fa.y - ra.y));
                    wop[u][t][1][WS - 1] = transpose8(pack_half2(fb.x - rb.x, fb.y - rb.y));
                }
            }
        }
#pragma unroll
        for (int t = 0; t < NT; t++) l[t] = add2(l[t], l1[t]), mn[t] = add2(mn[t], mn1[t]);
        // values: lane (g, c) holds dimensions 8 (VW g + w) .. + 7 of keys 2c, 2c+1, 2c+8, 2c+9
        uint32_t vw[KT][4][VW];
#pragma unroll
        for (int u = 0; u < KT; u++) {
            const uint8_t* vt = round + u * TB + 8 * DK + g * 4 * VW + c * DV;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint8_t* p = vt + ((j & 1) + (j >= 2 ? 8 : 0)) * (DV / 2);
                if constexpr (VW == 2) {
                    const uint2 x = *(const uint2*)p;
                    vw[u][j][0] = x.x, vw[u][j][1] = x.y;
                } else {
                    vw[u][j][0] = *(const uint32_t*)p;
                }
            }
        }
#pragma unroll
        for (int w = 0; w < VW; w++)
#pragma unroll
            for (int quarter = 0; quarter < 4; quarter++) {
                // dimensions 2 quarter (row g), 2 quarter + 1 (row g + 8)
                float z[F32 ? NT : 1][4];
#pragma unroll
                for (int u = 0; u < KT; u++) {
                    const uint32_t sel = quarter < 2 ? 0x5410 : 0x7632;
                    const uint32_t x = __byte_perm(vw[u][0][w], vw[u][1][w], sel) >> (quarter & 1 ? 8 : 0);
                    const uint32_t y = __byte_perm(vw[u][2][w], vw[u][3][w], sel) >> (quarter & 1 ? 8 : 0);
                    uint32_t a0 = x & 0x000f000fu, a1 = x & 0x00f000f0u, a2 = y & 0x000f000fu, a3 = y & 0x00f000f0u;
                    if (F32) a0 = code_mid(a0), a1 = code16_mid(a1), a2 = code_mid(a2), a3 = code16_mid(a3);
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        float* d = F32 ? z[F32 ? t : 0] : acc[t][4 * w + quarter];
                        if (F32 && u == 0) d[0] = d[1] = d[2] = d[3] = 0.f;
#pragma unroll
                        for (int term = 0; term < WS; term++) mma16816(d, a0, a1, a2, a3, wop[u][t][0][term], wop[u][t][1][term]);
                    }
                }
                if (F32)
#pragma unroll
                    for (int t = 0; t < NT; t++)
#pragma unroll
                        for (int j = 0; j < 4; j++) acc[t][4 * w + quarter][j] += z[F32 ? t : 0][j];
            }
    }
    asm volatile("cp.async.wait_group 0;\n" ::: "memory");
    __syncwarp();
    if (LONG && m > ROUNDS * KT) sums([&](int k, float x) { return (float)(past[k] + (Sum)x); });

    // this run's part of the unit: sums over the keys' lanes, 2^24 back
    const bool done = !part;
    const OutRows<T> to{out, a, rows.first, h, nrows};
#pragma unroll
    for (int t = 0; t < NT; t++) {
#pragma unroll
        for (int o = 4; o < 32; o *= 2) {
            l[t] = add2(l[t], __shfl_xor_sync(0xffffffffu, l[t], o));
            mn[t] = add2(mn[t], __shfl_xor_sync(0xffffffffu, mn[t], o));
        }
        const float2 l2 = unpair(l[t]), mn2 = unpair(mn[t]), M2 = unpair(nM[t]);
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const float lj = j ? l2.y : l2.x, mj = j ? mn2.y : mn2.x;
            const int y = 8 * t + 2 * c + j, x = b * 8 * NT + y;  // query row in the block, in the sequence
            const float norm = done ? (lj == 0.f ? 0.f : 1.f / lj) : 1.f;
#pragma unroll
            for (int w = 0; w < VW; w++) {
                float v[8];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    v[2 * k] = __fmaf_rn(acc[t][4 * w + k][j], F32 ? 1.f : 16777216.f, mj) * norm;
                    v[2 * k + 1] = __fmaf_rn(acc[t][4 * w + k][2 + j], F32 ? 1.f : 1048576.f, mj) * norm;
                }
                const int d0 = 8 * (VW * g + w);
                if (!done) store8(part + y * DV + d0, true, v);
                else if (x < nrows) store8(to.at(x) + d0, a.o_vec, v);
            }
            if (!done && g == 0) {
                part[8 * NT * DV + y] = j ? -M2.y : -M2.x;
                part[8 * NT * (DV + 1) + y] = lj;
            }
        }
    }
}

// Short units without sums over the sequences and without joins. SHARED: a
// CTA a unit, its warps share the tiles and join their parts in shared
// memory; else a warp a unit. blockIdx.x counts places, blockIdx.y kv heads.
template <int DK, int DV, int NT, typename T, bool SHARED>
__global__ void __launch_bounds__(32 * ATT_WARPS, AttendShape<DK, DV, NT, T>::CTAS)
    kv4_attend_whole_kernel(AttendArgs a, const T* __restrict__ q, T* __restrict__ out) {
    using Sh = AttendShape<DK, DV, NT, T>;
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (blockIdx.y == 0) zero_rest<DV>(a, out, blockIdx.x * ATT_WARPS + warp, gridDim.x * ATT_WARPS, lane);
    uint8_t* mine = smem + warp * (Sh::RING + Sh::QBYTES);
    uint2* qsm = (uint2*)(mine + Sh::RING);
    const int u = SHARED ? blockIdx.x : blockIdx.x * ATT_WARPS + warp, h = blockIdx.y;
    if (u >= a.places) return;
    int b;
    const int s = seq_of_place<NT>(a, u, lane, &b);
    if (s < 0) return;
    const SeqRows rows = seq_rows(a, s);
    if ((long long)b * 8 * NT >= (long long)rows.n * a.group.d) return;
    const Tiles tl = block_tiles<NT>(a, rows, b);
    if (!SHARED) {
        attend_part<DK, DV, NT, T, false>(a, q, out, s, h, b, rows, tl, 0, tl.n, mine, qsm, nullptr);
        return;
    }
    if constexpr (SHARED) {
        // as few warps as have a round each
        const int rounds = (tl.n + Sh::KT - 1) / Sh::KT, each = (rounds + ATT_WARPS - 1) / ATT_WARPS * Sh::KT;
        const int off = warp * each, m = min(each, tl.n - off), used = (tl.n + each - 1) / each;
        float* part = (float*)mine;  // over the ring
        if (m > 0) attend_part<DK, DV, NT, T, false>(a, q, out, s, h, b, rows, tl, off, m, mine, qsm, used == 1 ? nullptr : part);
        if (used == 1) return;
        __syncthreads();
        if (warp) return;
        PartRegs<DV> sum, more;
        sum.load(part, lane >> 2, lane & 3);
        for (int w = 1; w < used; w++) {
            more.load((const float*)(mine + w * (Sh::RING + Sh::QBYTES)), lane >> 2, lane & 3);
            sum.add(more);
        }
        sum.write(OutRows<T>{out, a, rows.first, h, rows.n * (int)a.group.d}, b * 8, lane >> 2, lane & 3);
    }
}

template <int DK, int DV, int NT, typename T>
__global__ void __launch_bounds__(32 * ATT_WARPS, AttendShape<DK, DV, NT, T>::CTAS)
    kv4_attend_kernel(AttendArgs a, const T* __restrict__ q, T* __restrict__ out) {
    using Sh = AttendShape<DK, DV, NT, T>;
    constexpr int PART = Sh::PART;
    constexpr bool MERGE = Sh::MERGE;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ long long sums[32 * ATT_WARPS + 1];
    __shared__ long long warp_sums[ATT_WARPS];
    __shared__ int4 cut_start[ATT_WARPS];   // the cut unit that starts in a warp's run: (sequence, kv head, block, 1), w = 0: none
    __shared__ int cut_rest[ATT_WARPS];     // the run begins inside a unit: 1, and ends it too: 2
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
    const int H = a.kv.heads, S = a.kv.seqs;
    const int warps = gridDim.x * ATT_WARPS, wid = blockIdx.x * ATT_WARPS + warp;

    zero_rest<DV>(a, out, wid, warps, lane);

    // the list's length, and its prefix at every chunk of `per` sequences
    const int per = (S + 32 * ATT_WARPS - 1) / (32 * ATT_WARPS);
    {
        long long mine = 0;
#pragma unroll 4
        for (int s = tid * per; s < min((tid + 1) * per, S); s++) mine += seq_work<NT>(a, seq_rows(a, s)) * H;
        long long incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const long long up = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += up;
        }
        if (lane == 31) warp_sums[warp] = incl;
        if (lane == 0) cut_start[warp] = make_int4(0, 0, 0, 0), cut_rest[warp] = 0;
        __syncthreads();
        for (int w = 0; w < warp; w++) incl += warp_sums[w];
        sums[tid + 1] = incl;
        if (tid == 0) sums[0] = 0;
        __syncthreads();
    }
    const long long total = sums[32 * ATT_WARPS];
    const long long share = max((total + warps - 1) / warps, (long long)ATT_MIN_SHARE);
    const long long begin = min(wid * share, total), end = min(begin + share, total);
    if (!MERGE && lane == 0) a.joins[wid] = make_int4(0, 0, 0, -1);

    uint8_t* mine = smem + warp * Sh::WARP_SMEM;
    float* first_part = (float*)(mine + Sh::RING + Sh::QBYTES);  // MERGE: a part of a unit that an earlier run begins
    float* last_part = (float*)mine;                // MERGE: of a unit that a later run ends, over the ring

    if (begin < end) {
        // the unit at `begin`
        int s;
        {
            int lo = 0, hi = 32 * ATT_WARPS;  // sums[lo] <= begin < sums[hi]
            while (hi - lo > 1) {
                const int mid = (lo + hi) / 2;
                if (sums[mid] <= begin) lo = mid;
                else hi = mid;
            }
            s = lo;
        }
        long long rem = begin - sums[s];
        s *= per;
        SeqRows rows = seq_rows(a, s);
        long long per_head = seq_work<NT>(a, rows);
        while (rem >= per_head * H) {
            rem -= per_head * H;
            rows = seq_rows(a, ++s);
            per_head = seq_work<NT>(a, rows);
        }
        int h = (int)(rem / per_head), b = 0;
        rem -= h * per_head;
        Tiles tl = block_tiles<NT>(a, rows, b);
        while (rem >= tl.n + ATT_UNIT_COST) {
            rem -= tl.n + ATT_UNIT_COST;
            tl = block_tiles<NT>(a, rows, ++b);
        }
        int at = (int)rem;  // place in the unit: its cost, then its tiles

        long long cur = begin;
        while (true) {
            const int span = (int)min((long long)(tl.n + ATT_UNIT_COST - at), end - cur);
            const int off = max(at - ATT_UNIT_COST, 0), m = max(at + span - ATT_UNIT_COST, 0) - off;
            const bool starts = off == 0, ends = off + m == tl.n, done = starts && ends;
            if (m) {
                float* part = MERGE ? (starts ? last_part : first_part) : a.parts + ((size_t)wid * 2 + (starts ? 1 : 0)) * PART;
                attend_part<DK, DV, NT, T, true>(a, q, out, s, h, b, rows, tl, off, m, mine, (uint2*)(mine + Sh::RING), done ? nullptr : part);
            }
            if (m && !done && lane == 0) {
                if (MERGE) {
                    if (starts) cut_start[warp] = make_int4(s, h, b, 1);
                    else cut_rest[warp] = ends ? 2 : 1;
                }
                if (starts) {
                    const long long last = (cur - at + tl.n + ATT_UNIT_COST - 1) / share;  // the warp that ends the unit
                    const int runner = MERGE ? blockIdx.x : wid, further = (int)((MERGE ? last / ATT_WARPS : last) - runner);
                    if (!MERGE) a.joins[wid] = make_int4(s, h, b, further);
                    else cut_start[warp].w = 1 + further;
                }
            }

            // the next unit
            cur += span;
            if (cur >= end) break;
            at = 0;
            if (++b * 8 * NT >= rows.n * (int)a.group.d) {
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

    if constexpr (MERGE) {
        __syncthreads();
        // A unit's parts in this CTA, from the warp where it starts (or warp
        // 0, if an earlier CTA has its start) to the one that ends it.
        auto slot = [&](int w, bool start) { return (const float*)(smem + w * Sh::WARP_SMEM + (start ? 0 : Sh::RING + Sh::QBYTES)); };
        auto chain = [&](bool start) {
            PartRegs<DV> sum, more;
            sum.load(slot(warp, start), g, c);
            bool ended = !start && cut_rest[warp] == 2;
            for (int w = warp + 1; w < ATT_WARPS && !ended && cut_rest[w]; w++) {
                more.load(slot(w, false), g, c);
                sum.add(more);
                ended = cut_rest[w] == 2;
            }
            if (start && ended) {
                const int4 u = cut_start[warp];
                const SeqRows rows = seq_rows(a, u.x);
                sum.write(OutRows<T>{out, a, rows.first, u.y, rows.n * (int)a.group.d}, u.z * 8, g, c);
                return false;
            }
            float* part = a.parts + ((size_t)blockIdx.x * 2 + (start ? 1 : 0)) * PART;
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int y = 2 * c + j;
#pragma unroll
                for (int k = 0; k < DV / 64; k++) store8(part + y * DV + (DV / 8) * g + 8 * k, true, sum.v[j] + 8 * k);
                if (g == 0) part[8 * DV + y] = sum.M[j], part[8 * (DV + 1) + y] = sum.l[j];
            }
            return true;
        };
        if (warp == 0 && cut_rest[0]) chain(false);
        if (cut_start[warp].w && chain(true) && lane == 0) {
            const int4 u = cut_start[warp];
            a.joins[blockIdx.x] = make_int4(u.x, u.y, u.z, u.w - 1);
        }
        // a CTA whose last cut unit ends here, or that has none, joins nothing
        if (tid == 0) {
            bool open = false;
            for (int w = 0; w < ATT_WARPS; w++) {
                if (open && cut_rest[w] != 1) open = false;
                if (cut_start[w].w) open = true;
            }
            if (!open) a.joins[blockIdx.x] = make_int4(0, 0, 0, -1);
        }
    }
}

// Blocks of 8 query rows, or of 16 where sequences bring many: the wider
// block halves the unpacking of codes a product, the narrower one splits over
// more warps and needs fewer registers. Measured (us, 8 against 16 rows): 5
// tokens of 6 heads a kv head, 256 sequences 50 and 52; 32 tokens of 4 heads
// 42 and 51; 512 tokens 393 and 339.
static int query_tiles(const nd_kv4* kv, int group) {
    return ((long long)kv->rows + kv->seqs - 1) / kv->seqs * group <= 256 ? 1 : 2;
}

// How a call is split:
// CUT   runs of equal work, units cut where they end, two kernels;
// WARP  a warp a unit, CTA  four warps a unit: units of few tiles.
// ROWS  blocks of 256 rows on tcgen05 (kv4_prefill.cu).
enum AttendMode { CUT, WARP, CTA, ROWS };

struct AttendPlan {
    int nt, ctas, places;
    AttendMode mode;
    size_t ws;
};

// Grid and workspace from what the host knows: the sizes, not the lengths.
static AttendPlan attend_plan(const nd_kv4* kv, int group, int type, int window, int sink) {
    AttendPlan p{};
    p.nt = query_tiles(kv, group);
    // tiles a unit can have: the table's, or those of the window (of 8 nt rows' tokens) and the sinks
    const long long table = (long long)kv->max_pages * (kv->page / KV4_TILE);
    long long tiles = table;
    if (window > 0) tiles = std::min(table, ((long long)window + 8 * p.nt + 2 * KV4_TILE) / KV4_TILE + (sink + KV4_TILE - 1LL) / KV4_TILE);
    const long long full = (long long)device_sm_count() * ATT_CTAS(p.nt, kv->dv);
    const long long further = (long long)kv->rows * group / (8 * p.nt);
    p.places = (int)(further + kv->seqs);
    const long long units = kv->heads * std::max<long long>(further, std::min(kv->seqs, kv->rows));  // as many as there are likely to be
    const long long most = kv->heads * (further + std::min(kv->seqs, kv->rows));
    p.mode = CUT;
    const long long rounds = (units + full - 1) / full;  // of a GPU full of CTAs
    if (p.nt == 1 && rounds <= 2 && rounds * tiles <= ATT_CTA_TILES && (rounds == 1 || tiles > ATT_WARP_TILES)) p.mode = CTA;
    else if (tiles <= ATT_WARP_TILES || (rounds > 1 && tiles <= ATT_WARP_MOST(kv->dv))) p.mode = WARP;
    if (p.mode == CUT && type != ND_F32 && (long long)kv->rows * group >= (long long)ATT_TC_ROWS * kv->seqs &&
        (long long)kv->heads * kv->rows * group / 8 * tiles >= ATT_TC_WORK(kv->dv)) {
        p.mode = ROWS;
        p.ws = prefill_ws_bytes(kv->dv, &p.ctas);
        return p;
    }
    const long long runs = (most * (tiles + ATT_UNIT_COST) + ATT_MIN_SHARE - 1) / ATT_MIN_SHARE;
    p.ctas = (int)std::max(1LL, std::min<long long>(full, (runs + ATT_WARPS - 1) / ATT_WARPS));
    const size_t runners = (size_t)p.ctas * (p.nt == 1 ? 1 : ATT_WARPS);
    p.ws = p.mode == CUT ? runners * (sizeof(int4) + 2 * sizeof(float) * 8 * p.nt * (kv->dv + 2)) : 0;
    return p;
}

template <int DK, int DV, int NT, typename T>
static void attend_launch(const AttendArgs& a0, const AttendPlan& plan, const void* q, void* out, void* ws, cudaStream_t st) {
    using Sh = AttendShape<DK, DV, NT, T>;
    AttendArgs a = a0;
    a.places = plan.places;
    auto check = [](cudaError_t e) {
        if (e != cudaSuccess) throw std::runtime_error(std::string("nd_op_kv4_attend: ") + cudaGetErrorString(e));
    };
    const char* what = "nd_op_kv4_attend";
    if (plan.mode == WARP) {
        allow_smem<kv4_attend_whole_kernel<DK, DV, NT, T, false>>(Sh::WHOLE_SMEM, what);
        kv4_attend_whole_kernel<DK, DV, NT, T, false><<<dim3((plan.places + ATT_WARPS - 1) / ATT_WARPS, a.kv.heads), 32 * ATT_WARPS, Sh::WHOLE_SMEM, st>>>(a, (const T*)q, (T*)out);
        return op_launched(what);
    }
    if constexpr (NT == 1)
        if (plan.mode == CTA) {
            allow_smem<kv4_attend_whole_kernel<DK, DV, NT, T, true>>(Sh::WHOLE_SMEM, what);
            kv4_attend_whole_kernel<DK, DV, NT, T, true><<<dim3(plan.places, a.kv.heads), 32 * ATT_WARPS, Sh::WHOLE_SMEM, st>>>(a, (const T*)q, (T*)out);
            return op_launched(what);
        }
    const int runners = plan.ctas * (Sh::MERGE ? 1 : ATT_WARPS);
    a.joins = (int4*)ws;
    a.parts = (float*)((char*)ws + (size_t)runners * sizeof(int4));
    allow_smem<kv4_attend_kernel<DK, DV, NT, T>>(Sh::SMEM, what);
    kv4_attend_kernel<DK, DV, NT, T><<<plan.ctas, 32 * ATT_WARPS, Sh::SMEM, st>>>(a, (const T*)q, (T*)out);
    op_launched(what);
    // launched early where the stream allows it; it waits for the first kernel's results
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(runners);
    cfg.blockDim = dim3(512);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = st ? 1 : 0;
    check(cudaLaunchKernelEx(&cfg, kv4_join_kernel<DV, NT, T>, (AttendArgs)a, (T*)out));
    add_launches(1);
}

template <int DK, int DV, typename T>
static void attend_nt(const AttendArgs& a, const AttendPlan& p, const void* q, void* out, void* ws, cudaStream_t st) {
    if (p.nt == 1) attend_launch<DK, DV, 1, T>(a, p, q, out, ws, st);
    else attend_launch<DK, DV, 2, T>(a, p, q, out, ws, st);
}

template <int DK, int DV>
static void attend_type(int type, const AttendArgs& a, const AttendPlan& p, const void* q, void* out, void* ws, cudaStream_t st) {
    if (type == ND_F32) attend_nt<DK, DV, float>(a, p, q, out, ws, st);
    else if (type == ND_F16) attend_nt<DK, DV, __half>(a, p, q, out, ws, st);
    else attend_nt<DK, DV, __nv_bfloat16>(a, p, q, out, ws, st);
}

static std::atomic<uint32_t> wait_rounds{tc::SPIN};

static int attend_group(const nd_kv4* kv, int q_heads, int window, int sink, const char* what) {
    auto fail = [&](const std::string& m) { throw std::runtime_error(std::string(what) + ": " + m); };
    if (q_heads < 1 || q_heads % kv->heads) fail("q_heads must be a multiple of heads");
    const int group = q_heads / kv->heads;
    if (group > 64) fail("more than 64 query heads a kv head");
    if ((long long)kv->rows * group > 0x7fffffffLL / 2) fail("too many rows");
    if (window < 0 || sink < 0) fail("window and sink must not be negative");
    return group;
}

}  // namespace nd

using namespace nd;

extern "C" {

unsigned long long nd_op_kv4_attend_ws(const nd_kv4* kv, int type, int q_heads, int window, int sink) {
    unsigned long long bytes = 0;
    op_call([&] {
        const char* what = "nd_op_kv4_attend_ws";
        kv4_args(kv, what);
        const int group = attend_group(kv, q_heads, window, sink, what);
        if (type != ND_F32 && type != ND_F16 && type != ND_BF16) throw std::runtime_error("nd_op_kv4_attend_ws: unknown type");
        OnDevice on(kv->device, what);
        bytes = attend_plan(kv, group, type, window, sink).ws;
    });
    return bytes;
}

unsigned nd_op_kv4_attend_wait_rounds(unsigned rounds) { return wait_rounds.exchange(rounds); }

int nd_op_kv4_attend(const nd_kv4* kv, int type, const void* q, long long q_row, long long q_head, int q_heads, float scale,
                     int window, int sink, void* out, long long o_row, long long o_head, void* ws, unsigned long long ws_bytes,
                     int flags, void* stream) {
    return op_call([&] {
        const char* what = "nd_op_kv4_attend";
        auto fail = [&](const std::string& m) { throw std::runtime_error(std::string(what) + ": " + m); };
        AttendArgs a{};
        a.kv = kv4_args(kv, what);
        const int group = attend_group(kv, q_heads, window, sink, what);
        if (!(fabsf(scale) <= FLT_MAX)) fail("scale must be finite");
        if (flags & ~ND_ZERO_REST) fail("unknown flags");
        if (a.kv.rows == 0) return;
        kv4_check_rows(what, type, q, q_row, q_head);
        kv4_check_out(what, type, out, o_row, o_head, a.kv.rows, q_heads, kv->dv);
        if ((uintptr_t)ws % 16) fail("the workspace must be 16-byte aligned");
        a.group = FastDiv(group), a.page_tiles = FastDiv(a.kv.page_tiles);
        a.q_row = q_row, a.q_head = q_head, a.o_row = o_row, a.o_head = o_head;
        a.window = window, a.sink = sink;
        a.scale_log2e = (float)((double)scale * 1.4426950408889634);
        a.q_vec = kv4_vec(type, q, q_row, q_head), a.o_vec = kv4_vec(type, out, o_row, o_head);
        a.zero_rest = flags & ND_ZERO_REST;
        a.wait_rounds = wait_rounds.load(std::memory_order_relaxed);
        OnDevice on(kv->device, what);
        const AttendPlan plan = attend_plan(kv, group, type, window, sink);
        if (plan.ws && (!ws || ws_bytes < plan.ws)) fail("the workspace is too small");
        cudaStream_t st = (cudaStream_t)stream;
        if (plan.mode == ROWS) prefill_launch(a, kv->dk, type, q, out, ws, st);
        else if (kv->dk == 48) attend_type<48, 64>(type, a, plan, q, out, ws, st);
        else if (kv->dk == 64) attend_type<64, 64>(type, a, plan, q, out, ws, st);
        else attend_type<128, 128>(type, a, plan, q, out, ws, st);
    });
}

}  // extern "C"
