// Attention over the paged 4-bit cache for many query rows a sequence
// (prompts): the same mathematics as kv4_attend.cu (see there) on the
// fifth-generation tensor cores, for bf16 and f16 rows.
//
// A CTA has 256 query rows of one kv head (two blocks of 128, tokens times
// the heads that share the kv head) and walks the visible keys 64 at a time:
//  - four warps read codes two stages ahead and write them to shared memory as
//    the f16 c - 8 (exact), keys as rows of K, values transposed, both in the
//    128-byte swizzle that the products read; so the unpacking is paid once
//    for 256 rows, and scales and minima stay in f32 beside them;
//  - one thread issues tcgen05.mma: S = Q C^T into tensor memory (two buffers
//    a block), O += P E with P from tensor memory;
//  - sixteen warps, two threads a row with 32 of the 64 keys each, turn S into
//    weights: x = sk_j S_ij + r_i mk_j, p = 2^(f_i x - M_i), w = p sv_j rounded
//    to f16 (in two terms for f16 rows) and written over S; the row's sums of
//    p and p mv stay in registers.
// Every PRE_SUMS stages O and the sums leave for the CTA's part in the workspace.
// M_i is raised only when a new exponent passes it by 4, and then O is
// rescaled in tensor memory; sv enters by its half stage's largest where that
// is near the others (PRE_SPREAD), so that w is at most 2^15 (ATT_TOP).
// The work is one list of equal runs as in kv4_attend.cu, cut at stages; cut
// units are joined by the same second kernel.
//
// Every wait is bounded; should one expire, the CTA's remaining rows are NaN, no
// further product is issued, and those under way are waited for.

#include "kernels.h"
#include "kv4_attend.cuh"
#include "kv4_host.h"
#include "tc.cuh"

namespace nd {

constexpr int PRE_KEYS = 64, PRE_STAGES = 3, PRE_THREADS = 768;
constexpr int PRE_NT = PRE_ROWS / 8;   // as block_tiles counts rows
// A half stage whose value scales lie within 2^PRE_SPREAD of one another takes
// the largest for all in its reference: weights lose that many bits of
// their range, not of their precision. Others are taken key by key, so that a
// large value that a row cannot see, or hardly weighs, costs it nothing.
constexpr float PRE_SPREAD = 4.f;
constexpr int PRE_UNIT_COST = 3;       // of beginning and ending a unit, in stages
// Stages after which a unit's sums leave tensor memory and registers and
// begin anew. The tensor cores truncate a running f32 sum at each product of 16
// keys: over 262,144 keys that cost f16 rows 3e-3 of the values.
constexpr int PRE_SUMS = 64;
// Registers of a thread: launched with 80 (the build checks that the compiler
// gave as many), then shared out by warpgroup (the rows' four, the operands',
// the issuer's), which sums to what was launched.
constexpr int PRE_REGS_LAUNCH = 80;
constexpr int PRE_REGS_ROWS = 88, PRE_REGS_CODES = 56, PRE_REGS_ISSUE = 72;
static_assert(4 * PRE_REGS_ROWS + PRE_REGS_CODES + PRE_REGS_ISSUE <= 6 * PRE_REGS_LAUNCH, "registers of the six warpgroups");

template <int DK, int DV, typename T>
struct PreShape {
    static constexpr int TB = kv4_tile_bytes(DK, DV);
    static constexpr int WS = std::is_same<T, __nv_bfloat16>::value ? 1 : 2;  // f16 terms of a weight
    static constexpr int ATOMS = DK > 64 ? 2 : 1;                             // 128-byte columns of a row of Q or K
    static constexpr int QB = 128 * 128 * ATOMS, KB = PRE_KEYS * 128 * ATOMS, VB = DV * 128;
    static constexpr int PART = PRE_ROWS * (DV + 2);
    static constexpr int SMEM = 1024 + 2 * QB + PRE_STAGES * (KB + VB);
};

// Of a stage's keys: scale, middle (minimum + 8 scales) of key and value;
// log2 of the value scale, less ATT_TOP; of each half the largest of these and
// how far above the smallest it lies; its four tiles' first
// positions and which of them exist; whether each block's rows all see all.
struct __align__(16) StageKeys {  // read by float4
    float ks[PRE_KEYS], km[PRE_KEYS], vs[PRE_KEYS], vm[PRE_KEYS];
    float lgs[PRE_KEYS], lg[2], spread[2];
    uint32_t have, whole;  // bits: tiles; blocks
    int k0[4];
};

// Four values of a row, by one store where `vec` says eight are aligned.
__device__ __forceinline__ void store4(__half* p, bool vec, float4 v) {
    if (vec) *(uint2*)p = make_uint2(pack_half2(v.x, v.y), pack_half2(v.z, v.w));
    else p[0] = __float2half_rn(v.x), p[1] = __float2half_rn(v.y), p[2] = __float2half_rn(v.z), p[3] = __float2half_rn(v.w);
}
__device__ __forceinline__ void store4(__nv_bfloat16* p, bool vec, float4 v) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
    if (vec) *(uint2*)p = make_uint2(*(const uint32_t*)&a, *(const uint32_t*)&b);
    else p[0] = a.x, p[1] = a.y, p[2] = b.x, p[3] = b.y;
}

__device__ __forceinline__ int stages_of(const Tiles& t) { return (t.n + 3) / 4; }

__device__ __forceinline__ long long pre_work(const AttendArgs& a, const SeqRows& r) {
    const int blocks = (r.n * (int)a.group.d + PRE_ROWS - 1) / PRE_ROWS;
    long long t = 0;
    for (int b = 0; b < blocks; b++) t += stages_of(block_tiles<PRE_NT>(a, r, b)) + PRE_UNIT_COST;
    return t;
}

template <int DK, int DV, typename T>
__global__ void __launch_bounds__(PRE_THREADS, 1) kv4_prefill_kernel(AttendArgs a, const T* __restrict__ q, T* __restrict__ out) {
    using Sh = PreShape<DK, DV, T>;
    constexpr int TB = Sh::TB, QB = Sh::QB, KB = Sh::KB, VB = Sh::VB, ST = PRE_STAGES;
    extern __shared__ uint8_t smem_raw[];
    __shared__ long long sums[PRE_THREADS + 1];
    __shared__ long long warp_sums[PRE_THREADS / 32];
    __shared__ __align__(16) StageKeys keys[ST];
    __shared__ __align__(8) uint64_t bars[2 * ST + 4 + 2 + 2 + 2];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag, late;
    // between the two warps of 32 rows: who wants a higher M, by stage parity;
    // the factors at the start, the sums at the end
    __shared__ int wish[2][2][8];
    __shared__ float wants[2][2][PRE_ROWS], half_l[PRE_ROWS], half_mn[PRE_ROWS];
    __shared__ float4 earlier[2][PRE_ROWS];  // a thread's M, sum p, sum p mv when its sums last left; they lie in its part's place
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    volatile int* abort = &abort_flag;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int H = a.kv.heads, S = a.kv.seqs, G = (int)a.group.d;
    const uint32_t base = (tc::smem_u32(smem_raw) + 1023u) & ~1023u;  // for the swizzle
    uint8_t* gbase = smem_raw + (base - tc::smem_u32(smem_raw));
    const uint32_t bar0 = tc::smem_u32(bars);
    auto full = [&](int s) { return bar0 + 8u * s; };
    auto empty = [&](int s) { return bar0 + 8u * (ST + s); };
    auto sfull = [&](int b, int buf) { return bar0 + 8u * (2 * ST + 2 * b + buf); };
    auto pready = [&](int b) { return bar0 + 8u * (2 * ST + 4 + b); };
    auto odone = [&](int b) { return bar0 + 8u * (2 * ST + 6 + b); };
    const uint32_t qready = bar0 + 8u * (2 * ST + 8), drained = bar0 + 8u * (2 * ST + 9);
    // a warp's wait: all its lanes go on, or none
    auto warp_wait = [&](uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, tc::bar_wait(bar, parity, abort, a.wait_rounds)) != 0; };

    zero_rest<DV>(a, out, blockIdx.x * (PRE_THREADS / 32) + warp, gridDim.x * (PRE_THREADS / 32), lane);
    if (tid == 0) {
        for (int s = 0; s < ST; s++) tc::bar_init(full(s), 4), tc::bar_init(empty(s), 1);
        for (int b = 0; b < 2; b++) {
            tc::bar_init(sfull(b, 0), 1), tc::bar_init(sfull(b, 1), 1);
            tc::bar_init(pready(b), 8), tc::bar_init(odone(b), 1);
        }
        tc::bar_init(qready, 16);
        tc::bar_init(drained, 1);
        abort_flag = late = 0;
        a.joins[blockIdx.x] = make_int4(0, 0, 0, -1);
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == 20) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(tc::smem_u32(&tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    // the list's length, and its prefix at every chunk of `per` sequences
    const int per = (S + PRE_THREADS - 1) / PRE_THREADS;
    {
        long long mine = 0;
        for (int s = tid * per; s < min((tid + 1) * per, S); s++) mine += pre_work(a, seq_rows(a, s)) * H;
        long long incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const long long up = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += up;
        }
        if (lane == 31) warp_sums[warp] = incl;
        tc::fence_before();
        __syncthreads();
        tc::fence_after();
        for (int w = 0; w < warp; w++) incl += warp_sums[w];
        sums[tid + 1] = incl;
        if (tid == 0) sums[0] = 0;
        __syncthreads();
    }
    const uint32_t tmem = tmem_slot;
    const long long total = sums[PRE_THREADS];
    const long long share = max((total + gridDim.x - 1) / gridDim.x, (long long)(2 * PRE_UNIT_COST));
    const long long begin = min(blockIdx.x * share, total), end = min(begin + share, total);

    // Calls f(s, h, b, rows, tiles, first stage, stages, its number in this
    // CTA, stages before it) for each part of a unit in this CTA's run. All
    // roles walk the same parts.
    auto for_parts = [&](auto&& f) {
        if (begin >= end) return;
        int s;
        {
            int lo = 0, hi = PRE_THREADS;  // sums[lo] <= begin < sums[hi]
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
        long long per_head = pre_work(a, rows);
        while (rem >= per_head * H) {
            rem -= per_head * H;
            rows = seq_rows(a, ++s);
            per_head = pre_work(a, rows);
        }
        int h = (int)(rem / per_head), b = 0;
        rem -= h * per_head;
        Tiles tl = block_tiles<PRE_NT>(a, rows, 0);
        while (rem >= stages_of(tl) + PRE_UNIT_COST) {
            rem -= stages_of(tl) + PRE_UNIT_COST;
            tl = block_tiles<PRE_NT>(a, rows, ++b);
        }
        int at = (int)rem, part = 0, it = 0;
        for (long long cur = begin;;) {
            const int ns = stages_of(tl), span = (int)min((long long)(ns + PRE_UNIT_COST - at), end - cur);
            const int off = max(at - PRE_UNIT_COST, 0), m = max(at + span - PRE_UNIT_COST, 0) - off;
            if (m) {
                f(s, h, b, rows, tl, off, m, part, it, cur - at + ns + PRE_UNIT_COST - 1);
                part++, it += m;
            }
            cur += span;
            if (cur >= end) break;
            at = 0;
            if (++b * PRE_ROWS >= rows.n * G) {
                b = 0;
                if (++h == H) {
                    h = 0;
                    do rows = seq_rows(a, ++s);
                    while (rows.n == 0);
                }
            }
            tl = block_tiles<PRE_NT>(a, rows, b);
        }
    };

    if (warp < 16) {
        // ---- two threads a query row: block, half of the keys, row
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(PRE_REGS_ROWS));
        const int blk = warp >> 3, half = warp >> 2 & 1, row = tid & 127, pair_no = blk * 4 + (warp & 3);
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t scol = tmem + lanes + blk * 256 + 32 * half, ocol = tmem + lanes + blk * 256 + 128 + DV / 2 * half;
        uint8_t* qs = gbase + blk * QB;
        auto pair_sync = [&]() { asm volatile("bar.sync %0, 64;\n" ::"r"(1 + pair_no) : "memory"); };
        bool ok = true;
        for_parts([&](int s, int h, int b, const SeqRows& rows, const Tiles& tl, int off, int m, int part_no, int it0, long long last) {
            const int nrows = rows.n * G, x0 = b * PRE_ROWS + blk * 128, x = x0 + row;
            const bool active = x0 < nrows, on = x < nrows;
            const int tok = a.group(min(x, nrows - 1));
            // the rows' queries as f16 of 2^14 at the largest, in the order in
            // which codes are unpacked: 0 4 1 5 2 6 3 7 of every eight. The
            // warp has sixteen rows, LQ lanes a row, all loads under way at
            // once; each row's factors go to its threads through shared memory
            float f = 0.f, r = 0.f;
            if (active) {
                constexpr int LQ = DK > 64 ? 16 : 8, PER = 32 / LQ, TURNS = 16 / PER;
                const int sub = lane % LQ, y0 = 32 * (warp & 3) + 16 * half + lane / LQ;
                float v[TURNS][8];
#pragma unroll
                for (int t = 0; t < TURNS; t++) {
                    const int xq = x0 + y0 + PER * t, tq = a.group(min(xq, nrows - 1));
                    const bool have_q = xq < nrows && 8 * sub < DK;
#pragma unroll
                    for (int i = 0; i < 8; i++) v[t][i] = 0.f;
                    if (have_q)
                        load8(q + (long long)(rows.first + tq) * a.q_row + (long long)(h * G + xq - tq * G) * a.q_head + 8 * sub, a.q_vec, v[t]);
                }
                const float sign = a.scale_log2e < 0.f ? -1.f : 1.f;
#pragma unroll
                for (int t = 0; t < TURNS; t++) {
                    const int y = y0 + PER * t;
                    float top = 0.f, sum = 0.f;
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        top = fmaxf(top, fabsf(v[t][i]));
                        sum += v[t][i];
                    }
#pragma unroll
                    for (int o = 1; o < LQ; o *= 2) {
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                        sum += __shfl_xor_sync(0xffffffffu, sum, o);
                    }
                    const bool bad = !(top <= FLT_MAX && sum == sum);  // an infinity, a NaN
                    const int e = min(max((int)(__float_as_uint(top) >> 23) - 127, -100), 127);
                    const float up = bad ? 0.f : sign * __uint_as_float((uint32_t)(14 - e + 127) << 23);
                    if (8 * sub < DK) {
#pragma unroll
                        for (int i = 0; i < 8; i++) v[t][i] = bad ? 0.f : v[t][i] * up;
                        *(uint4*)(qs + (sub / 8) * (128 * 128) + y * 128 + ((sub % 8) ^ (y & 7)) * 16) =
                            make_uint4(pack_half2(v[t][0], v[t][4]), pack_half2(v[t][1], v[t][5]), pack_half2(v[t][2], v[t][6]), pack_half2(v[t][3], v[t][7]));
                    }
                    if (sub == 0) {
                        // exponents are f x: f positive, so that the largest x has the largest
                        const float nan = __uint_as_float(0x7fc00000u);
                        half_l[blk * 128 + y] = bad ? nan : fmaxf(fabsf(a.scale_log2e) * __uint_as_float((uint32_t)(e - 14 + 127) << 23), 1e-37f);
                        half_mn[blk * 128 + y] = bad ? nan : sum * up;
                    }
                }
                tc::fence_async_smem();
                pair_sync();
                f = half_l[blk * 128 + row], r = half_mn[blk * 128 + row];
                pair_sync();
            }
            tc::fence_before();
            __syncwarp();
            if (lane == 0) tc::bar_arrive(qready);

            const int hi = on ? (int)min(max(rows.pos0 + tok, -1LL), 0x7fffffffLL) : -1;
            const f32x2 f2 = pair(f, f), r2 = pair(r, r);
            float M = ATT_LOW;
            f32x2 l2 = 0, mn2 = 0;
            const bool starts = off == 0, ends = off + m == stages_of(tl), done = starts && ends;
            float* part = a.parts + ((size_t)blockIdx.x * 2 + (starts ? 1 : 0)) * Sh::PART;
            // a thread's own dimensions of its row there
            float* own = part + (size_t)(blk * 128 + row) * DV + DV / 2 * half;

#pragma unroll 1
            for (int i = 0; i < m; i++) {
                const int k = it0 + i, slot = k % ST, buf = k & 1;
                if (ok) ok = warp_wait(sfull(blk, buf), (k >> 1) & 1) && warp_wait(full(slot), (k / ST) & 1);
                if (active) {
                    // both warps of the rows come here whether or not a wait has failed
                    tc::fence_after();
                    const StageKeys& sk = keys[slot];
                    float xs[32];
                    tc::ld32(scol + buf * 64, xs);
                    tc::ld_wait32(xs);
                    const bool whole = sk.whole >> blk & 1;
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        const float4 ks = *(const float4*)&sk.ks[32 * half + j], km = *(const float4*)&sk.km[32 * half + j];
                        const float2 y = unpair(fma2(pair(xs[j], xs[j + 1]), pair(ks.x, ks.y), mul2(r2, pair(km.x, km.y))));
                        const float2 z = unpair(fma2(pair(xs[j + 2], xs[j + 3]), pair(ks.z, ks.w), mul2(r2, pair(km.z, km.w))));
                        xs[j] = y.x, xs[j + 1] = y.y, xs[j + 2] = z.x, xs[j + 3] = z.y;
                    }
                    if (__builtin_expect(!whole, 0)) {
#pragma unroll
                        for (int j = 0; j < 32; j++) {
                            const int tile = 2 * half + j / 16, key = sk.k0[tile] + j % 16;
                            if (!((sk.have >> tile & 1) && key <= hi && (a.window <= 0 || key > hi - a.window || key < a.sink))) xs[j] = -INFINITY;
                        }
                    }
                    float t4[4] = {xs[0], xs[1], xs[2], xs[3]};
#pragma unroll
                    for (int j = 4; j < 32; j++) t4[j & 3] = fmaxf(t4[j & 3], xs[j]);
                    const float top = fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3]));
                    float want = __fmaf_rn(top, f, sk.lg[half]);
                    if (__builtin_expect(sk.spread[half] > PRE_SPREAD, 0)) {
                        want = -INFINITY;
#pragma unroll
                        for (int j = 0; j < 32; j += 4) {
                            const float4 lg = *(const float4*)&sk.lgs[32 * half + j];
                            want = fmaxf(fmaxf(want, fmaxf(__fmaf_rn(xs[j], f, lg.x), __fmaf_rn(xs[j + 1], f, lg.y))),
                                         fmaxf(__fmaf_rn(xs[j + 2], f, lg.z), __fmaf_rn(xs[j + 3], f, lg.w)));
                        }
                    }
                    const bool any = __any_sync(0xffffffffu, want > M + 4.f);
                    if (lane == 0) wish[buf][half][pair_no] = any;
                    if (any) wants[buf][half][blk * 128 + row] = want;
                    pair_sync();
                    const bool other = wish[buf][half ^ 1][pair_no];
                    if (__builtin_expect(any || other, 0)) {
                        float to = M;
                        if (any && want > M + 4.f) to = want;
                        if (other) {
                            const float w = wants[buf][half ^ 1][blk * 128 + row];
                            if (w > M + 4.f) to = fmaxf(to, w);
                        }
                        const float scale = ex2(M - to);
                        M = to;
                        l2 = mul2(l2, pair(scale, scale)), mn2 = mul2(mn2, pair(scale, scale));
                        if (i > 0) {
                            if (ok) ok = warp_wait(odone(blk), (k - 1) & 1);
                            tc::fence_after();
                            if (ok)
#pragma unroll 1
                                for (int c = 0; c < DV / 2; c += 16) {
                                    float o[16];
                                    tc::ld16(ocol + c, o);
                                    tc::ld_wait16(o);
#pragma unroll
                                    for (int j = 0; j < 16; j++) o[j] *= scale;
                                    tc::st16(ocol + c, (const uint32_t*)o);
                                }
                        }
                    }
                    const f32x2 nM = pair(-M, -M);
                    // weights over the half's own scores
                    auto weigh = [&](bool clean) {
                        uint32_t w[16 * Sh::WS];
                        f32x2 l1 = 0, mn1 = 0;  // this stage's: small terms meet before a large sum
#pragma unroll
                        for (int j = 0; j < 32; j += 4) {
                            const float4 vs = *(const float4*)&sk.vs[32 * half + j], vm = *(const float4*)&sk.vm[32 * half + j];
#pragma unroll
                            for (int t = 0; t < 2; t++) {
                                const float2 xx = make_float2(xs[j + 2 * t], xs[j + 2 * t + 1]);
                                const float2 e = unpair(fma2(pair(xx.x, xx.y), f2, nM));
                                f32x2 p = pair(ex2(e.x), ex2(e.y));
                                f32x2 s2 = t ? pair(vs.z, vs.w) : pair(vs.x, vs.y), m2 = t ? pair(vm.z, vm.w) : pair(vm.x, vm.y);
                                if (clean) {  // a masked place, or its query, may hold NaN or infinity
                                    p = pair(xx.x == -INFINITY ? 0.f : ex2(e.x), xx.y == -INFINITY ? 0.f : ex2(e.y));
                                    const float2 sf = unpair(s2), mf = unpair(m2);
                                    s2 = pair(xx.x == -INFINITY ? 0.f : sf.x, xx.y == -INFINITY ? 0.f : sf.y);
                                    m2 = pair(xx.x == -INFINITY ? 0.f : mf.x, xx.y == -INFINITY ? 0.f : mf.y);
                                }
                                l1 = add2(l1, p);
                                mn1 = fma2(p, m2, mn1);
                                const float2 v = unpair(mul2(p, s2));
                                const uint32_t hw = pack_half2(v.x, v.y);
                                w[j / 2 + t] = hw;
                                if (Sh::WS == 2) {
                                    const float2 back = unpack_half2(hw);
                                    w[16 * (Sh::WS - 1) + j / 2 + t] = pack_half2(v.x - back.x, v.y - back.y);
                                }
                            }
                        }
                        l2 = add2(l2, l1), mn2 = add2(mn2, mn1);
                        if constexpr (Sh::WS == 2) tc::st32(scol + buf * 64, w);
                        else tc::st16(scol + buf * 64, w);
                    };
                    if (__builtin_expect(whole, 1)) weigh(false);
                    else weigh(true);
                    tc::st_wait();
                    tc::fence_before();
                }
                // the last product's phase is seen before this stage's weights
                // are announced: a parity tells only neighbouring phases apart,
                // here of odone and for the issuing thread of pready
                if (ok && i > 0) ok = warp_wait(odone(blk), (k - 1) & 1);
                if (__builtin_expect(i > 0 && i % PRE_SUMS == 0, 0) && active && ok) {
                    // the product of this stage starts from zero
                    tc::fence_after();
                    const bool first = i == PRE_SUMS;
                    float4 e = first ? make_float4(M, 0.f, 0.f, 0.f) : earlier[half][blk * 128 + row];
                    const float scale = ex2(e.x - M);
#pragma unroll 1
                    for (int c = 0; c < DV / 2; c += 16) {
                        float o[16];
                        tc::ld16(ocol + c, o);
                        tc::ld_wait16(o);
#pragma unroll
                        for (int j = 0; j < 16; j += 4) {
                            float4 v = make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]);
                            if (!first) {
                                const float4 w = *(const float4*)(own + c + j);
                                v.x = __fmaf_rn(w.x, scale, v.x), v.y = __fmaf_rn(w.y, scale, v.y);
                                v.z = __fmaf_rn(w.z, scale, v.z), v.w = __fmaf_rn(w.w, scale, v.w);
                            }
                            *(float4*)(own + c + j) = v;
                        }
                    }
                    // of this stage too, which O has not
                    const float2 lp = unpair(l2), mp = unpair(mn2);
                    e.y = __fmaf_rn(e.y, scale, lp.x + lp.y), e.z = __fmaf_rn(e.z, scale, mp.x + mp.y);
                    l2 = mn2 = 0;
                    e.x = M;
                    earlier[half][blk * 128 + row] = e;
                    tc::fence_before();
                }
                __syncwarp();
                if (lane == 0) tc::bar_arrive(pready(blk));
            }

            // the last product, and the result or this CTA's part of it
            if (ok) ok = warp_wait(odone(blk), (it0 + m - 1) & 1);
            // what another role did after giving up may have reached this part
            __threadfence_block();
            if (__any_sync(0xffffffffu, *abort)) ok = false;
            if (active) {
                tc::fence_after();
                const float2 lp = unpair(l2), mp = unpair(mn2);
                float l = lp.x + lp.y, mn = mp.x + mp.y, scale = 0.f;
                const bool more = m > PRE_SUMS && ok;
                if (more) {
                    const float4 e = earlier[half][blk * 128 + row];
                    scale = ex2(e.x - M);
                    l = __fmaf_rn(e.y, scale, l), mn = __fmaf_rn(e.z, scale, mn);
                }
                if (!ok) l = __uint_as_float(0x7fc00000u);
                const int y = blk * 128 + row;
                // the halves' sums, each row's in one order
                if (half) half_l[y] = l, half_mn[y] = mn;
                pair_sync();
                if (!half) {
                    l += half_l[y], mn += half_mn[y];
                    half_l[y] = l, half_mn[y] = mn;
                }
                pair_sync();
                l = half_l[y], mn = half_mn[y];
                const float norm = done ? (l == 0.f ? 0.f : 1.f / l) : 1.f;
                const OutRows<T> to{out, a, rows.first, h, nrows};
                // by way of the queries' shared memory, which this block's
                // products are done with, so that rows leave as whole lines:
                // a thread a row has 32 of them open at once, which took 8 to
                // 12 thousand cycles a part
                constexpr int CR = DK > 64 ? 32 : 16, QUADS = CR / 4;  // dimensions a turn
                float4* stage = (float4*)(qs + ((warp & 3) * 2 + half) * (32 * CR * 4));
#pragma unroll 1
                for (int c = 0; c < DV / 2; c += CR) {
#pragma unroll
                    for (int u = 0; u < CR; u += 16) {
                        float o[16];
                        tc::ld16(ocol + c + u, o);
                        tc::ld_wait16(o);
                        if (more)
#pragma unroll
                            for (int j = 0; j < 16; j += 4) {
                                const float4 w = *(const float4*)(own + c + u + j);
                                o[j] = __fmaf_rn(w.x, scale, o[j]), o[j + 1] = __fmaf_rn(w.y, scale, o[j + 1]);
                                o[j + 2] = __fmaf_rn(w.z, scale, o[j + 2]), o[j + 3] = __fmaf_rn(w.w, scale, o[j + 3]);
                            }
#pragma unroll
                        for (int j = 0; j < 16; j += 4)
                            stage[lane * QUADS + (((u + j) / 4) ^ (lane & (QUADS - 1)))] =
                                make_float4((o[j] + mn) * norm, (o[j + 1] + mn) * norm, (o[j + 2] + mn) * norm, (o[j + 3] + mn) * norm);
                    }
                    __syncwarp();
#pragma unroll
                    for (int t = 0; t < QUADS; t++) {
                        const int yy = t * (32 / QUADS) + lane / QUADS, quad = lane % QUADS;
                        const float4 v = stage[yy * QUADS + (quad ^ (yy & (QUADS - 1)))];
                        const int yb = blk * 128 + 32 * (warp & 3) + yy, xr = b * PRE_ROWS + yb, d = DV / 2 * half + c + 4 * quad;
                        if (!done) *(float4*)(part + (size_t)yb * DV + d) = v;
                        else if (xr < nrows) store4(to.at(xr) + d, a.o_vec, v);
                    }
                    __syncwarp();
                }
                if (!done && !half) part[PRE_ROWS * DV + y] = M, part[PRE_ROWS * (DV + 1) + y] = l;
                tc::fence_before();
                // the queries' place is written again by any of the block's warps
                asm volatile("bar.sync %0, 256;\n" ::"r"(9 + blk) : "memory");
            }
            if (starts && !ends && tid == 0) a.joins[blockIdx.x] = make_int4(s, h, b, (int)(last / share - blockIdx.x));
        });
    } else if (warp < 20) {
        // ---- codes to operands
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(PRE_REGS_CODES));
        const int t = tid - 512, half = t >> 6, key = t & 63, w4 = warp - 16;
        constexpr int KW = DK / 16, VWW = DV / 32;  // words of a half key row; of a quarter value row
        bool ok = true;
        for_parts([&](int s, int h, int b, const SeqRows& rows, const Tiles& tl, int off, int m, int part_no, int it0, long long last) {
            const int first = 4 * off, n = min(4 * m, tl.n - first);  // tiles of this part
            const int32_t* trow = a.kv.table + (size_t)s * a.kv.table_stride;
            const uint8_t* head = a.kv.pool + (size_t)h * a.kv.page_tiles * TB;
            const long long len = rows.pos0 + rows.n;
            // tiles wholly inside every row's span of a block need no masks
            int all_hi[2], all_lo[2];
#pragma unroll
            for (int blk = 0; blk < 2; blk++) {
                const int x0 = min(b * PRE_ROWS + blk * 128, rows.n * G - 1), x1 = min(b * PRE_ROWS + blk * 128 + 128, rows.n * G) - 1;
                all_hi[blk] = (int)min(max(rows.pos0 + a.group(x0), -1LL), 0x7fffffffLL) - 15;
                all_lo[blk] = a.window > 0 ? (int)min(max(rows.pos0 + a.group(max(x1, 0)) - a.window, -1LL), 0x7fffffffLL) : -1;
            }
            auto fetch = [&](int i) -> unsigned long long {  // the i-th tile's address, 0: no such page
                if (i >= n) return 0;
                const int tile = tl.at(first + i), p = a.page_tiles(tile);
                const int page = p < a.kv.max_pages ? __ldg(trow + p) : -1;
                if (page < 0 || page >= a.kv.num_pages) return 0;
                return (unsigned long long)(head + (size_t)page * a.kv.page_stride + (size_t)(tile - p * a.kv.page_tiles) * TB);
            };
            unsigned long long src = fetch(lane), src_next = fetch(32 + lane);
            uint32_t kw[KW], vw[2][VWW], kp = 0, vp = 0, have = 0;
            bool held = false;  // this thread's key exists
            auto load = [&](int i) {  // stage i's words
                if (i && (i & 7) == 0) src = src_next, src_next = fetch(4 * i + 32 + lane);
                const unsigned long long ka = __shfl_sync(0xffffffffu, src, (4 * i + (key >> 4)) & 31);
                const unsigned long long va = __shfl_sync(0xffffffffu, src, (4 * i + (lane >> 3)) & 31);
                have = __ballot_sync(0xffffffffu, src != 0) >> (4 * i & 31) & 15;
#pragma unroll
                for (int w = 0; w < KW; w++) kw[w] = 0x88888888u;  // c - 8 = 0
#pragma unroll
                for (int w = 0; w < VWW; w++) vw[0][w] = vw[1][w] = 0x88888888u;
                kp = vp = 0, held = false;
                if (ka) {
                    const uint8_t* p = (const uint8_t*)ka + (key & 15) * (DK / 2) + half * (DK / 4);
                    if constexpr (DK == 48) {
#pragma unroll
                        for (int w = 0; w < KW; w++) kw[w] = __ldg((const uint32_t*)p + w);
                    } else {
#pragma unroll
                        for (int w = 0; w < KW; w += 4) {
                            const uint4 x = __ldg((const uint4*)p + w / 4);
                            kw[w] = x.x, kw[w + 1] = x.y, kw[w + 2] = x.z, kw[w + 3] = x.w;
                        }
                    }
                    if (half == 0 && tl.at(first + 4 * i + (key >> 4)) * (long long)KV4_TILE + (key & 15) < len) {
                        const uint8_t* pp = (const uint8_t*)ka + 8 * (DK + DV) + 4 * (key & 15);
                        kp = __ldg((const uint32_t*)pp), vp = __ldg((const uint32_t*)(pp + 64)), held = true;
                    }
                }
                if (va) {
                    const uint8_t* p = (const uint8_t*)va + 8 * DK + (2 * lane & 15) * (DV / 2) + w4 * (DV / 8);
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        if constexpr (VWW == 4) {
                            const uint4 x = __ldg((const uint4*)(p + u * (DV / 2)));
                            vw[u][0] = x.x, vw[u][1] = x.y, vw[u][2] = x.z, vw[u][3] = x.w;
                        } else {
                            const uint2 x = __ldg((const uint2*)(p + u * (DV / 2)));
                            vw[u][0] = x.x, vw[u][1] = x.y;
                        }
                    }
                }
            };
            load(0);
#pragma unroll 1
            for (int i = 0; i < m; i++) {
                const int k = it0 + i, slot = k % ST;
                if (ok && k >= ST) ok = warp_wait(empty(slot), ((k / ST) - 1) & 1);
                uint8_t* ks = gbase + 2 * QB + slot * (KB + VB);
                uint8_t* vs = ks + KB;
#pragma unroll
                for (int w = 0; w < KW; w++) {  // eight dimensions: 16 bytes of the key's row
                    const int c = half * KW + w;
                    const uint32_t x = kw[w], y = x >> 8;
                    *(uint4*)(ks + (c / 8) * (PRE_KEYS * 128) + key * 128 + ((c % 8) ^ (key & 7)) * 16) =
                        make_uint4(code_mid(x & 0x000f000fu), code16_mid(x & 0x00f000f0u), code_mid(y & 0x000f000fu), code16_mid(y & 0x00f000f0u));
                }
#pragma unroll
                for (int w = 0; w < VWW; w++)
#pragma unroll
                    for (int q4 = 0; q4 < 4; q4++) {  // dimensions 2 q4, 2 q4 + 1 of keys 2 lane, 2 lane + 1
                        const uint32_t x = __byte_perm(vw[0][w], vw[1][w], q4 < 2 ? 0x5410 : 0x7632) >> (q4 & 1 ? 8 : 0);
                        const int d = w4 * (DV / 4) + 8 * w + 2 * q4;
                        uint8_t* p = vs + (lane & 3) * 4;
                        *(uint32_t*)(p + d * 128 + (((lane >> 2) ^ (d & 7)) * 16)) = code_mid(x & 0x000f000fu);
                        *(uint32_t*)(p + (d + 1) * 128 + (((lane >> 2) ^ ((d + 1) & 7)) * 16)) = code16_mid(x & 0x00f000f0u);
                    }
                if (half == 0) {
                    StageKeys& sk = keys[slot];
                    const float2 kf = unpack_half2(kp), vf = unpack_half2(vp);
                    sk.ks[key] = kf.x, sk.km[key] = __fmaf_rn(8.f, kf.x, kf.y);
                    sk.vs[key] = vf.x, sk.vm[key] = __fmaf_rn(8.f, vf.x, vf.y);
                    const float lg = lg2(fmaxf(vf.x, 5.9604645e-8f)) - ATT_TOP;
                    sk.lgs[key] = lg;
                    // positions that do not exist (their scales are zeros) leave the spread alone
                    float most = held ? lg : -INFINITY, least = held ? lg : INFINITY;
#pragma unroll
                    for (int o = 16; o; o /= 2) {
                        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
                        least = fminf(least, __shfl_xor_sync(0xffffffffu, least, o));
                    }
                    if (lane == 0) sk.lg[w4] = most, sk.spread[w4] = most - least;
                    if (t == 0) {
                        uint32_t see = have == 15 ? 3 : 0;
#pragma unroll
                        for (int u = 0; u < 4; u++) {
                            const int k0 = tl.at(first + 4 * i + u) * KV4_TILE;
                            sk.k0[u] = k0;
#pragma unroll
                            for (int blk = 0; blk < 2; blk++)
                                if (!(k0 <= all_hi[blk] && (k0 > all_lo[blk] || k0 + 15 < a.sink))) see &= ~(1u << blk);
                        }
                        sk.have = have, sk.whole = see;
                    }
                }
                tc::fence_async_smem();
                __syncwarp();
                if (lane == 0) tc::bar_arrive(full(slot));
                if (i + 1 < m) load(i + 1);
            }
        });
    } else {
        // ---- the products: an elected lane of the first of four warps issues
        // them. What a product takes is the same in all lanes and known to be
        // (shuffled), and differs by constants from step to step.
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(PRE_REGS_ISSUE));
        bool ok = true;
        bool issued = false;
        const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0), q_lo = tc::sw128_lo(__shfl_sync(0xffffffffu, base, 0));
        if (warp == 20) for_parts([&](int s, int h, int b, const SeqRows& rows, const Tiles& tl, int off, int m_, int part_no, int it0_, long long last) {
            const int m = __shfl_sync(0xffffffffu, m_, 0), it0 = __shfl_sync(0xffffffffu, it0_, 0);
            const bool both = __shfl_sync(0xffffffffu, b * PRE_ROWS + 128 < rows.n * G, 0);
            if (ok) ok = warp_wait(qready, part_no & 1);
            auto scores = [&](int k) {
                const int slot = k % ST;
                if (ok) ok = warp_wait(full(slot), (k / ST) & 1);
                if (!ok) return;
                tc::fence_after();
                const uint32_t k_lo = q_lo + ((2 * QB + slot * (KB + VB)) >> 4), d = tm + (k & 1) * 64;
                issued = true;
                if (tc::elect()) {
#pragma unroll
                    for (int c = 0; c < DK / 16; c++)
                        tc::mma_ss(d, q_lo + c / 4 * (128 * 128 >> 4) + c % 4 * 2, k_lo + c / 4 * (PRE_KEYS * 128 >> 4) + c % 4 * 2, tc::f16_idesc(PRE_KEYS), c > 0);
                    tc::commit(sfull(0, k & 1));
                    if (both)
#pragma unroll
                        for (int c = 0; c < DK / 16; c++)
                            tc::mma_ss(d + 256, q_lo + (QB >> 4) + c / 4 * (128 * 128 >> 4) + c % 4 * 2, k_lo + c / 4 * (PRE_KEYS * 128 >> 4) + c % 4 * 2,
                                       tc::f16_idesc(PRE_KEYS), c > 0);
                    tc::commit(sfull(1, k & 1));
                }
                __syncwarp();
            };
            scores(it0);
#pragma unroll 1
            for (int i = 0; i < m && ok; i++) {
                const int k = it0 + i, slot = k % ST;
                if (i + 1 < m) scores(k + 1);
                const uint32_t v_lo = q_lo + ((2 * QB + slot * (KB + VB) + KB) >> 4), p = tm + (k & 1) * 64;
#pragma unroll
                for (int blk = 0; blk < 2; blk++) {
                    if (ok) ok = warp_wait(pready(blk), k & 1);
                    if (!ok) break;
                    tc::fence_after();
                    if (tc::elect()) {
                        if (blk == 0 || both)
#pragma unroll
                            for (int term = 0; term < Sh::WS; term++)
#pragma unroll
                                for (int c = 0; c < PRE_KEYS / 16; c++)
                                    tc::mma_ts(tm + blk * 256 + 128, p + blk * 256 + c / 2 * 32 + term * 16 + c % 2 * 8, v_lo + c * 2, tc::f16_idesc(DV),
                                               term > 0 || c > 0 ? 1u : (uint32_t)(i % PRE_SUMS != 0));
                        tc::commit(odone(blk));
                        if (blk == 1) tc::commit(empty(slot));
                    }
                    __syncwarp();
                }
            }
        });
        // Every product issued, by the same lane each time, is over before its
        // memory is freed, also where a wait has expired: this one has its own bound.
        if (warp == 20 && issued) {
            if (tc::elect()) tc::commit(drained);
            __syncwarp();
            tc::bar_wait(drained, 0, &late);
        }
    }
    tc::fence_before();
    __syncthreads();
    if (warp == 20) {
        tc::fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512) : "memory");
    }
}

size_t prefill_ws_bytes(int dv, int* ctas) {
    *ctas = device_sm_count();
    return (size_t)*ctas * (sizeof(int4) + 2 * sizeof(float) * PRE_ROWS * (dv + 2));
}

template <int DK, int DV, typename T>
static void launch(const AttendArgs& a0, const void* q, void* out, void* ws, cudaStream_t st) {
    using Sh = PreShape<DK, DV, T>;
    AttendArgs a = a0;
    const int ctas = device_sm_count();
    a.joins = (int4*)ws;
    a.parts = (float*)((char*)ws + (size_t)ctas * sizeof(int4));
    auto check = [](cudaError_t e) {
        if (e != cudaSuccess) throw std::runtime_error(std::string("nd_op_kv4_attend: ") + cudaGetErrorString(e));
    };
    allow_smem<kv4_prefill_kernel<DK, DV, T>>(Sh::SMEM, "nd_op_kv4_attend");
    kv4_prefill_kernel<DK, DV, T><<<ctas, PRE_THREADS, Sh::SMEM, st>>>(a, (const T*)q, (T*)out);
    op_launched("nd_op_kv4_attend");
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(ctas, 8);
    cfg.blockDim = dim3(512);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = st ? 1 : 0;
    check(cudaLaunchKernelEx(&cfg, kv4_join_kernel<DV, PRE_NT, T>, AttendArgs(a), (T*)out));
    add_launches(1);
}

template <typename T>
static void launch_dk(const AttendArgs& a, int dk, const void* q, void* out, void* ws, cudaStream_t st) {
    if (dk == 48) launch<48, 64, T>(a, q, out, ws, st);
    else if (dk == 64) launch<64, 64, T>(a, q, out, ws, st);
    else launch<128, 128, T>(a, q, out, ws, st);
}

void prefill_launch(const AttendArgs& a, int dk, int type, const void* q, void* out, void* ws, cudaStream_t st) {
    if (type == ND_F16) launch_dk<__half>(a, dk, q, out, ws, st);
    else launch_dk<__nv_bfloat16>(a, dk, q, out, ws, st);
}

}  // namespace nd
