// Drafted tokens against the target's probabilities (nd_op_verify).
//
// With p_i = softmax(logits_i / temperature) and q_i the draft's probabilities,
// the drafted token x_i stands while u_i q_i(x_i) < p_i(x_i); the first that
// falls is replaced by a draw from max(p_i - q_i, 0), and after the last a
// token is drawn from p. What matters here is that a draw is an index that a
// rounding near a border would change: sums, exponentials and comparisons
// that decide are in f64. Nearly all of the work is not: a row's maximum is
// exact in any order, its sum of exponentials is taken from f32 terms first,
// and a comparison closer than 1e-4 to its border is decided again with the
// sum in f64. That first sum is off by less than 1e-5 whatever V: 2^-22 of each
// ex2 and 2^-22 |x| of its argument, where |x| 2^x is below 0.6 or x up to
// VF_SLACK; five roundings of 2^-24 where a thread adds 16 terms, f64 from
// there; as much as a term again where parts meet, and at each rescaling, of
// which at most 11 leave a part that counts. Only the one row a sequence draws
// from is summed in f64 throughout.
//
// Two kernels: one takes every row's statistics (one read of the logits, which
// bounds the large calls: a CTA a row, or several where rows are few), the
// second, a cluster of CTAs a sequence, decides and draws. There every warp
// has a run of the drawn row: the runs' sums meet through the cluster's
// shared memory, each CTA adds them up in order, and the warp whose run holds
// the place walks it 32 values at a time.
//
// Measured (us, GPU alone; 256 sequences of up to 7 drafts, 16384 f32 logits):
// one kernel with a CTA a row 236; two kernels 64, the second waiting for
// its f64 terms one after another; with terms in batches of four without
// branches 53, batches of eight whose places need no checks 45. Runs of 512 on
// four CTAs instead of 1024 on two took 4 more. An exponential of fewer f64
// steps (a table of 2^(j/16)) gained nothing: issue and latency bound it.

#include <cooperative_groups.h>

#include <cfloat>

#include "kv4_host.h"

namespace nd {

namespace cg = cooperative_groups;

constexpr int VF_MAX_DRAFT = 64, VF_MAX_SEQS = 1 << 20, VF_MAX_V = 1 << 30;
constexpr int VF_STATS = 256;        // threads of the first kernel
constexpr int VF_CHUNK = 4096;       // logits a CTA of it takes at a time
constexpr int VF_MAX_PARTS = 32;
// CTAs that rows are cut for: four an SM. A constant, so that a workspace's
// size does not depend on which device is current when it is asked for.
constexpr int VF_FILL = 4 * 148;
constexpr float VF_SLACK = 2.f;      // of an exponent of two
constexpr int VF_DRAW = 256, VF_WARPS = VF_DRAW / 32;  // of the second
// Runs are made this short where eight CTAs can; a warp keeps its run's terms
// up to this length, two CTAs an SM; and up to this where a CTA has an SM to
// itself, if the grid is at most two rounds of that. Past it they are computed
// twice (us, twice and kept: 16 sequences of 130,000 logits 65, 36; 32 of
// 100,000 66, 44; 32 of 130,000 72, 68; but 128 of 130,000 124, 167).
constexpr int VF_RUN = 1024, VF_CACHE = 1696, VF_CACHE_ALONE = 3392;
constexpr int BATCH = 8;  // that a lane takes at a time
constexpr float LOG2E = 1.4426950408889634f;

// Of a row, or a part of it: the largest logit; its first place where the
// draw is greedy, else 0 (-1: no distribution, a NaN is there); sum exp((l -
// top) / temperature) where it is not greedy.
struct RowStats {
    float top;
    int at;
    double sum;
};

struct VerifyArgs {
    long long l_seq, l_row, q_seq, q_row;
    const int32_t* draft;   // [seqs][T]
    const int32_t* counts;  // [seqs] or NULL
    const float* u;         // [seqs][T + 1]
    const float* temp;      // [seqs]
    const float* q;         // or NULL
    int seqs, T, V, parts;
    bool l_vec, kept;  // a drawn row's terms are
    RowStats* stats;             // [seqs][T + 1][parts]
    int32_t *tokens, *accepted;  // [seqs][T + 1], [seqs]
    float* probs;                // [seqs][T + 1]
};

__device__ __forceinline__ float vf_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ int drafts_of(const VerifyArgs& a, int s) { return a.counts ? min(max(__ldg(a.counts + s), 0), a.T) : a.T; }

struct Temperature {
    bool greedy;
    double inv;
    float pre, scale2;  // of an exponent of two: pre is 1, or 2^64 where LOG2E / t is no f32
    __device__ explicit Temperature(float t) {
        greedy = !(t > 0.f);
        t = fminf(t, FLT_MAX);  // an infinite one: the limit, where -infinity still has no part
        inv = greedy ? 1.0 : 1.0 / (double)t;
        pre = !greedy && t < 1e-37f ? 18446744073709551616.f : 1.f;
        scale2 = greedy ? LOG2E : LOG2E / (t * pre);
    }
    // d / t as an exponent of two
    __device__ __forceinline__ float two(float d) const { return d * pre * scale2; }
};

template <typename T>
__global__ void __launch_bounds__(VF_STATS) verify_stats_kernel(VerifyArgs a, const T* __restrict__ logits) {
    constexpr int PER = 16 / sizeof(T), LOADS = VF_CHUNK / VF_STATS / PER, N = LOADS * PER;
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    const int r = blockIdx.x / a.parts, part = blockIdx.x % a.parts, s = r / (a.T + 1), i = r % (a.T + 1), tid = threadIdx.x;
    if (i > drafts_of(a, s)) return;
    const Temperature tp(__ldg(a.temp + s));
    const bool greedy = tp.greedy;
    const T* row = logits + s * a.l_seq + i * a.l_row;
    const int chunks = (a.V + VF_CHUNK - 1) / VF_CHUNK, per = (chunks + a.parts - 1) / a.parts;
    const int lo = min(part * per, chunks), hi = min(lo + per, chunks);
    // The sum is against `ref`, which follows the largest logit only when that
    // is 2^VF_SLACK ahead: each time the sum loses 2^-22 of what is left of it,
    // which is little. A chunk's terms meet in f32, chunks in f64, so that the
    // error does not grow with V.
    float top = -INFINITY, ref = -INFINITY;
    double sum = 0.0;
    int at = a.V;
    bool nan = false;
    uint4 raw[LOADS];  // the next chunk, where 16-byte loads reach all of it
    auto whole = [&](int ch) { return a.l_vec && ch < hi && (ch + 1) * VF_CHUNK <= a.V; };
    auto fetch = [&](int ch) {
        if (whole(ch))
#pragma unroll
            for (int k = 0; k < LOADS; k++) raw[k] = __ldg((const uint4*)(row + ch * VF_CHUNK) + k * VF_STATS + tid);
    };
    fetch(lo);
    for (int ch = lo; ch < hi; ch++) {
        float x[N];
        const int base = ch * VF_CHUNK;
        if (whole(ch)) {
#pragma unroll
            for (int k = 0; k < LOADS; k++) {
                const uint32_t w[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    if constexpr (sizeof(T) == 4) {
                        x[4 * k + j] = __uint_as_float(w[j]);
                    } else {
                        const T* h = (const T*)&w[j];
                        x[8 * k + 2 * j] = (float)h[0], x[8 * k + 2 * j + 1] = (float)h[1];
                    }
                }
            }
            fetch(ch + 1);
        } else {  // the same places one by one
#pragma unroll
            for (int j = 0; j < N; j++) {
                const int p = base + (j / PER * VF_STATS + tid) * PER + j % PER;
                x[j] = p < a.V ? (float)row[p] : -INFINITY;
            }
        }
        if (greedy) {  // the place; NaN by itself
#pragma unroll
            for (int j = 0; j < N; j++) {
                nan |= x[j] != x[j];
                if (x[j] > top) top = x[j], at = base + (j / PER * VF_STATS + tid) * PER + j % PER;
            }
        } else {  // the sum, which a NaN spoils, as +infinity does
            float m = top;
#pragma unroll
            for (int j = 0; j < N; j++) m = fmaxf(m, x[j]);
            if (m == -INFINITY) {
#pragma unroll
                for (int j = 0; j < N; j++) nan |= x[j] != x[j];
                continue;
            }
            top = m;
            if (tp.two(m - ref) > VF_SLACK) sum *= (double)vf_ex2(tp.two(ref - m)), ref = m;  // ref = -infinity: sum is 0
            float part[4];
#pragma unroll
            for (int j = 0; j < N; j++) {
                const float e = vf_ex2(tp.two(x[j] - ref));
                part[j & 3] = j < 4 ? e : part[j & 3] + e;
            }
            sum += (double)((part[0] + part[1]) + (part[2] + part[3]));
        }
    }
    if (!greedy) nan |= sum != sum, at = top > -INFINITY ? 0 : a.V;
    // the block's largest, its first place, the sum against it
    __shared__ float tops[VF_STATS / 32];
    __shared__ int ats[VF_STATS / 32];
    __shared__ double sums[VF_STATS / 32];
    const int lane = tid & 31, warp = tid >> 5;
    float m = top;
#pragma unroll
    for (int o = 16; o; o /= 2) {
        const float om = __shfl_xor_sync(0xffffffffu, m, o);
        const int oa = __shfl_xor_sync(0xffffffffu, at, o);
        if (om > m || (om == m && oa < at)) m = om, at = oa;
        nan |= __shfl_xor_sync(0xffffffffu, (int)nan, o) != 0;
    }
    if (lane == 0) tops[warp] = m, ats[warp] = nan ? -1 : at;
    __syncthreads();
    m = tops[0], at = ats[0], nan = at < 0;
#pragma unroll
    for (int w = 1; w < VF_STATS / 32; w++) {
        nan |= ats[w] < 0;
        if (tops[w] > m || (tops[w] == m && ats[w] < at)) m = tops[w], at = ats[w];
    }
    double z = top == -INFINITY ? 0.0 : sum * (double)vf_ex2(tp.two(ref - m));
#pragma unroll
    for (int o = 16; o; o /= 2) z += __shfl_xor_sync(0xffffffffu, z, o);
    if (lane == 0) sums[warp] = z;
    __syncthreads();
    if (tid == 0) {
        z = 0.0;
        for (int w = 0; w < VF_STATS / 32; w++) z += sums[w];
        a.stats[blockIdx.x] = RowStats{m, nan ? -1 : at, z};
    }
}

// exp(x) for x <= 0 (NaN stays), without branches, so that the terms of a run
// overlap: x = k ln 2 + r with ln 2 in two parts (Cody and Waite; the first
// has 40 bits, k times it is exact), Taylor's series to r^13 (|r| <= 0.35:
// 4e-18 left), times 2^k. Within 2^-52 of itself; below e^-708, 0.
__device__ __forceinline__ double exp_below(double x) {
    const bool tiny = x < -708.0;
    const double y = tiny ? -708.0 : x;
    const double t = __fma_rn(y, 1.4426950408889634, 6755399441055744.0);  // 1.5 * 2^52: its low bits hold k
    const double k = t - 6755399441055744.0;
    const double r = __fma_rn(k, 1.7239444525614835e-13, __fma_rn(k, -0.6931471805601177, y));
    double p = 1.6059043836821613e-10;
    p = __fma_rn(p, r, 2.08767569878681e-09);  // 1 / 12!
    p = __fma_rn(p, r, 2.505210838544172e-08);  // 1 / 11!
    p = __fma_rn(p, r, 2.755731922398589e-07);  // 1 / 10!
    p = __fma_rn(p, r, 2.7557319223985893e-06);  // 1 / 9!
    p = __fma_rn(p, r, 2.48015873015873e-05);  // 1 / 8!
    p = __fma_rn(p, r, 0.0001984126984126984);  // 1 / 7!
    p = __fma_rn(p, r, 0.001388888888888889);  // 1 / 6!
    p = __fma_rn(p, r, 0.008333333333333333);  // 1 / 5!
    p = __fma_rn(p, r, 0.041666666666666664);  // 1 / 4!
    p = __fma_rn(p, r, 0.16666666666666666);  // 1 / 3!
    p = __fma_rn(p, r, 0.5);
    p = __fma_rn(p, r, 1.0);
    p = __fma_rn(p, r, 1.0);
    const double e = p * __hiloint2double((__double2loint(t) + 1023) << 20, 0);
    return tiny ? 0.0 : e;
}

template <typename T>
__device__ __forceinline__ double term(const T* row, int j, float top, double inv) {
    return exp_below(((double)(float)row[j] - (double)top) * inv);
}

__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
    for (int o = 16; o; o /= 2) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}

// A row's statistics from its parts, in their order; at < 0 where it is no
// distribution. For a whole warp.
__device__ __forceinline__ RowStats join_stats(const RowStats* parts, int n, const Temperature& tp, int lane) {
    RowStats r{-INFINITY, 0x7fffffff, 0.0};
    if (lane < n) r = parts[lane];
    float m = r.top;
    int at = r.at;
    bool nan = r.at < 0;
#pragma unroll
    for (int o = 16; o; o /= 2) {
        const float om = __shfl_xor_sync(0xffffffffu, m, o);
        const int oa = __shfl_xor_sync(0xffffffffu, at, o);
        if (om > m || (om == m && oa < at)) m = om, at = oa;
        nan |= __shfl_xor_sync(0xffffffffu, (int)nan, o) != 0;
    }
    RowStats out{m, nan || m == -INFINITY ? -1 : at, 0.0};
    out.sum = warp_sum(r.top == -INFINITY ? 0.0 : r.sum * (double)vf_ex2(tp.two(r.top - m)));
    return out;
}

// Values a warp takes of a row that `runs` warps share.
__host__ __device__ __forceinline__ int run_of(int V, int runs) { return ((V + runs - 1) / runs + 31) / 32 * 32; }

template <typename T>
__global__ void __launch_bounds__(VF_DRAW) verify_draw_kernel(VerifyArgs a, const T* __restrict__ logits) {
    cg::cluster_group cluster = cg::this_cluster();
    const int C = cluster.num_blocks(), rank = cluster.block_rank(), s = blockIdx.x / C;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    __shared__ RowStats rows[VF_MAX_DRAFT + 1];
    __shared__ int verdict[VF_MAX_DRAFT + 1];  // 0 refused, 1 accepted, 2 too close to say
    __shared__ double probs[VF_MAX_DRAFT + 1];
    __shared__ double sums[2][VF_WARPS];  // by warp: of its run's terms, of its residuals
    __shared__ double all[8 * VF_WARPS];  // those of every run
    extern __shared__ double cache_all[];
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    const int T_ = a.T, V = a.V, n = drafts_of(a, s);
    const Temperature tp(__ldg(a.temp + s));
    const float* u = a.u + (size_t)s * (T_ + 1);
    const T* l0 = logits + s * a.l_seq;

    // p of a drafted token and its verdict, given the row's sum
    auto judge = [&](int i, const RowStats& st, bool sure, double* p) -> int {
        *p = 0.0;
        const int x = __ldg(a.draft + (size_t)s * T_ + i);
        if (st.at < 0 || x < 0 || x >= V) return 0;
        const double uq = (double)__ldg(u + i) * (a.q ? (double)__ldg(a.q + s * a.q_seq + i * a.q_row + x) : 1.0);
        if (tp.greedy) {
            *p = x == st.at;
            return uq < *p;
        }
        const double e = term(l0 + i * a.l_row, x, st.top, tp.inv);
        *p = e / st.sum;
        if (!sure && fabs(uq * st.sum - e) <= 1e-4 * (fabs(uq * st.sum) + e)) return 2;
        return uq < *p;
    };
    for (int i = warp; i <= n; i += VF_WARPS) {
        const RowStats st = join_stats(a.stats + ((size_t)s * (T_ + 1) + i) * a.parts, a.parts, tp, lane);
        if (lane == 0) {
            rows[i] = st;
            if (i < n) verdict[i] = judge(i, st, false, &probs[i]);
        }
    }
    __syncthreads();
    int kept = 0;
    for (; kept < n; kept++) {
        int v = verdict[kept];
        if (v == 2) {  // the same for every thread: the row's sum in f64
            RowStats st = rows[kept];
            double z = 0.0;
            for (int j = tid; j < V; j += VF_DRAW) z += term(l0 + kept * a.l_row, j, st.top, tp.inv);
            z = warp_sum(z);
            if (lane == 0) sums[0][warp] = z;
            __syncthreads();
            st.sum = 0.0;
            for (int w = 0; w < VF_WARPS; w++) st.sum += sums[0][w];
            double p;
            v = judge(kept, st, true, &p);
            __syncthreads();
            if (tid == 0) probs[kept] = p;
        }
        if (v == 0) break;
    }
    __syncthreads();

    const size_t o = (size_t)s * (T_ + 1);
    auto finish = [&](int token, double p) { a.tokens[o + kept] = token, a.probs[o + kept] = (float)p; };
    if (rank == 0) {
        for (int i = tid; i <= T_; i += VF_DRAW) {
            if (i == kept) continue;
            a.tokens[o + i] = i < kept ? __ldg(a.draft + (size_t)s * T_ + i) : -1;
            a.probs[o + i] = i < kept ? (float)probs[i] : 0.f;
        }
        if (tid == 0) a.accepted[s] = kept;
    }
    const RowStats st = rows[kept];
    if (st.at < 0 || tp.greedy) {
        // no distribution; or one at st.at, which what q takes from it leaves the only token
        if (rank == 0 && tid == 0) finish(st.at, st.at < 0 ? 0.0 : 1.0);
        return;
    }

    // the drawn row: this warp's run, its terms kept where they fit
    const T* row = l0 + kept * a.l_row;
    const float* q = kept < n && a.q ? a.q + s * a.q_seq + kept * a.q_row : nullptr;
    const int gone = kept < n && !a.q ? __ldg(a.draft + (size_t)s * T_ + kept) : -1;
    const int runs = C * VF_WARPS, run = rank * VF_WARPS + warp;
    const int per = run_of(V, runs), lo = (int)min((long long)run * per, (long long)V), hi = min(lo + per, V);
    double* cache = cache_all + warp * per;  // the run's terms, where they fit
    const bool fits = a.kept;
    // BATCH values 32 apart at a time, without branches between them, so that
    // their loads and their chains of products overlap; what is left one by one
    double mine = 0.0;
    int j = lo + lane;
    for (; j - lane + 32 * BATCH <= hi; j += 32 * BATCH) {
        const T* x = row + j;
        double e[BATCH];
#pragma unroll
        for (int k = 0; k < BATCH; k++) e[k] = (double)(float)x[32 * k];
#pragma unroll
        for (int k = 0; k < BATCH; k++) e[k] = exp_below((e[k] - (double)st.top) * tp.inv);
#pragma unroll
        for (int k = 0; k < BATCH; k++) {
            if (fits) cache[j - lo + 32 * k] = e[k];
            mine += e[k];
        }
    }
    for (; j < hi; j += 32) {
        const double e = term(row, j, st.top, tp.inv);
        if (fits) cache[j - lo] = e;
        mine += e;
    }
    mine = warp_sum(mine);
    if (lane == 0) sums[0][warp] = mine;
    // every run's sum from its CTA: lane l of each warp gets those of runs
    // EACH l .., what lies before them, and the whole
    constexpr int EACH = 8 * VF_WARPS / 32;
    double v[EACH], ahead;
    auto gather = [&](int which) {
        cluster.sync();
        if (tid < 8 * VF_WARPS) all[tid] = tid < runs ? cluster.map_shared_rank(&sums[which][0], tid / VF_WARPS)[tid % VF_WARPS] : 0.0;
        __syncthreads();
        double own = 0.0;
#pragma unroll
        for (int k = 0; k < EACH; k++) v[k] = all[EACH * lane + k], own += v[k];
        double incl = own;
#pragma unroll
        for (int k = 1; k < 32; k *= 2) {
            const double up = __shfl_up_sync(0xffffffffu, incl, k);
            if (lane >= k) incl += up;
        }
        ahead = __shfl_up_sync(0xffffffffu, incl, 1);
        if (lane == 0) ahead = 0.0;
        return __shfl_sync(0xffffffffu, incl, 31);
    };
    const double iz = 1.0 / gather(0);
    bool whole = false;  // p itself, where the residual is all zero
    // what can be drawn of value j, of which the term is e
    auto rest = [&](int j, double e, float qj) {
        const double r = e * iz - (double)qj;
        return r < 0.0 || (j == gone && !whole) ? 0.0 : r;
    };
    auto weight = [&](int j) {
        return rest(j, fits ? cache[j - lo] : term(row, j, st.top, tp.inv), q && !whole ? __ldg(q + j) : 0.f);
    };
    double total;
    while (true) {
        mine = 0.0;
        j = lo + lane;
        for (; j - lane + 32 * BATCH <= hi; j += 32 * BATCH) {
            double e[BATCH];
            float qj[BATCH];
#pragma unroll
            for (int k = 0; k < BATCH; k++) qj[k] = q && !whole ? __ldg(q + j + 32 * k) : 0.f;
#pragma unroll
            for (int k = 0; k < BATCH; k++) e[k] = fits ? cache[j - lo + 32 * k] : term(row, j + 32 * k, st.top, tp.inv);
#pragma unroll
            for (int k = 0; k < BATCH; k++) mine += rest(j + 32 * k, e[k], qj[k]);
        }
        for (; j < hi; j += 32) mine += weight(j);
        mine = warp_sum(mine);
        if (lane == 0) sums[1][warp] = mine;
        total = gather(1);
        if (total != 0.0 || whole) break;
        whole = true;
        cluster.sync();  // the others have read the sums
    }
    if (total > 0.0) {
        // the first run in which the running sum passes the target, or where
        // none does (u is 1) the last that has something to draw
        const double target = fmin(fmax((double)__ldg(u + T_), 0.0), 1.0) * total;
        double cum = ahead, before = 0.0, last_before = 0.0;
        int at = -1, last = -1;
#pragma unroll
        for (int k = 0; k < EACH; k++) {
            if (v[k] > 0.0) {
                last = EACH * lane + k, last_before = cum;
                if (at < 0 && cum + v[k] > target) at = last, before = cum;
            }
            cum += v[k];
        }
        const uint32_t hits = __ballot_sync(0xffffffffu, at >= 0), some = __ballot_sync(0xffffffffu, last >= 0);
        const bool passed = hits != 0;
        const int from = passed ? __ffs(hits) - 1 : 31 - __clz(some);
        at = __shfl_sync(0xffffffffu, passed ? at : last, from);
        before = __shfl_sync(0xffffffffu, passed ? before : last_before, from);
        if (at == run) {
            // the lanes share the run, per / 32 values each in order, and all
            // of them the values of the one that holds the place
            auto prefix = [&](double w, double* incl) {
                *incl = w;
#pragma unroll
                for (int k = 1; k < 32; k *= 2) {
                    const double up = __shfl_up_sync(0xffffffffu, *incl, k);
                    if (lane >= k) *incl += up;
                }
            };
            const int each = per / 32;
            double own = 0.0, incl;
            bool some = false;
#pragma unroll 4
            for (int j = lo + lane * each, end = min(j + each, hi); j < end; j++) {
                const double w = weight(j);
                own += w, some |= w > 0.0;
            }
            prefix(own, &incl);
            // should the sums' last bits differ, the last lane that has something
            const uint32_t past = __ballot_sync(0xffffffffu, some && passed && before + incl > target);
            const int from = past ? __ffs(past) - 1 : 31 - __clz(__ballot_sync(0xffffffffu, some));
            before += __shfl_sync(0xffffffffu, incl - own, from);
            int token = -1;
            for (int j0 = lo + from * each, end = min(j0 + each, hi); j0 < end; j0 += 32) {
                const double w = j0 + lane < end ? weight(j0 + lane) : 0.0;
                prefix(w, &incl);
                const uint32_t any = __ballot_sync(0xffffffffu, w > 0.0);
                const uint32_t hit = __ballot_sync(0xffffffffu, w > 0.0 && past && before + incl > target);
                if (any) token = j0 + 31 - __clz(any);
                if (hit) {
                    token = j0 + __ffs(hit) - 1;
                    break;
                }
                before += __shfl_sync(0xffffffffu, incl, 31);
            }
            if (lane == 0) finish(token, term(row, token, st.top, tp.inv) * iz);
        }
    } else if (rank == 0 && tid == 0) {
        finish(-1, 0.0);
    }
    cluster.sync();  // no CTA leaves while others read its sums
}

static int verify_parts(int seqs, int T, int V) {
    // few rows: enough CTAs for the GPU, a chunk each at least
    const long long rows = (long long)seqs * (T + 1), chunks = (V + VF_CHUNK - 1) / VF_CHUNK;
    return (int)std::max(1LL, std::min({chunks, (long long)VF_MAX_PARTS, VF_FILL / rows}));
}

static unsigned long long verify_ws(int seqs, int T, int V) {
    return (unsigned long long)seqs * (T + 1) * verify_parts(seqs, T, V) * sizeof(RowStats);
}

template <typename T>
static void verify_launch(const VerifyArgs& a, const void* logits, int ctas, cudaStream_t st) {
    auto check = [](cudaError_t e) {
        if (e != cudaSuccess) throw std::runtime_error(std::string("nd_op_verify: ") + cudaGetErrorString(e));
    };
    verify_stats_kernel<T><<<(unsigned)a.seqs * (a.T + 1) * a.parts, VF_STATS, 0, st>>>(a, (const T*)logits);
    op_launched("nd_op_verify");
    constexpr int MOST = VF_WARPS * VF_CACHE_ALONE * sizeof(double);
    allow_smem<verify_draw_kernel<T>>(MOST, "nd_op_verify");
    const int per = run_of(a.V, ctas * VF_WARPS);
    VerifyArgs b(a);
    b.kept = per <= ((long long)a.seqs * ctas <= 2 * device_sm_count() ? VF_CACHE_ALONE : VF_CACHE);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)a.seqs * ctas);
    cfg.blockDim = dim3(VF_DRAW);
    cfg.dynamicSmemBytes = b.kept ? VF_WARPS * per * sizeof(double) : 0;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = ctas, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = st ? 2 : 1;
    check(cudaLaunchKernelEx(&cfg, verify_draw_kernel<T>, b, (const T*)logits));
    add_launches(1);
}

}  // namespace nd

using namespace nd;

extern "C" {

unsigned long long nd_op_verify_ws(int seqs, int T, int V) {
    return seqs < 1 || seqs > VF_MAX_SEQS || T < 0 || T > VF_MAX_DRAFT || V < 1 || V > VF_MAX_V ? 0 : verify_ws(seqs, T, V);
}

int nd_op_verify(int device, int type, const void* logits, long long l_seq, long long l_row, const int* draft,
                 const int* counts, const float* u, const float* temperature, const float* q, long long q_seq, long long q_row,
                 int seqs, int T, int V, int* tokens, int* accepted, float* probs, void* ws, unsigned long long ws_bytes,
                 void* stream) {
    return op_call([&] {
        const char* what = "nd_op_verify";
        auto fail = [&](const std::string& m) { throw std::runtime_error(std::string(what) + ": " + m); };
        if (type != ND_F32 && type != ND_F16 && type != ND_BF16) fail("unknown type");
        if (seqs < 1 || seqs > VF_MAX_SEQS || T < 0 || T > VF_MAX_DRAFT || V < 1 || V > VF_MAX_V)
            fail("needs 1 to 2^20 sequences, 0 to 64 drafted tokens, 1 <= V <= 2^30");
        if (!logits || !u || !temperature || !tokens || !accepted || !probs || (T && !draft)) fail("null pointer");
        const int e = type == ND_F32 ? 4 : 2;
        if ((uintptr_t)logits % e || (uintptr_t)q % 4) fail("logits and q must be aligned to their types");
        if (l_seq < 0 || l_row < 0 || q_seq < 0 || q_row < 0) fail("negative strides");
        if (!ws || (uintptr_t)ws % 16 || ws_bytes < verify_ws(seqs, T, V)) fail("the workspace is too small or not 16-byte aligned");
        VerifyArgs a{};
        a.l_seq = l_seq, a.l_row = l_row, a.q_seq = q_seq, a.q_row = q_row;
        a.draft = draft, a.counts = counts, a.u = u, a.temp = temperature, a.q = T ? q : nullptr;
        a.seqs = seqs, a.T = T, a.V = V, a.parts = verify_parts(seqs, T, V);
        a.l_vec = (uintptr_t)logits % 16 == 0 && l_seq * e % 16 == 0 && l_row * e % 16 == 0;
        a.stats = (RowStats*)ws;
        a.tokens = tokens, a.accepted = accepted, a.probs = probs;
        OnDevice on(device, what);
        // CTAs a drawn row: until a warp's terms fit its cache, or while they do not fill the GPU and runs are not short
        int ctas = 1;
        while (ctas < 8 && V > 1024 * ctas && (V > VF_WARPS * VF_RUN * ctas || seqs * ctas < 2 * device_sm_count())) ctas *= 2;
        cudaStream_t st = (cudaStream_t)stream;
        if (type == ND_F32) verify_launch<float>(a, logits, ctas, st);
        else if (type == ND_F16) verify_launch<__half>(a, logits, ctas, st);
        else verify_launch<__nv_bfloat16>(a, logits, ctas, st);
    });
}

}  // extern "C"
