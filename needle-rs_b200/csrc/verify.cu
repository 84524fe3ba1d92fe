// Drafted tokens against the target's probabilities (nd_op_verify).
//
// With p_i = softmax(logits_i / temperature) and q_i the draft's probabilities,
// the drafted token x_i stands while u_i q_i(x_i) < p_i(x_i); the first that
// falls is replaced by a draw from max(p_i - q_i, 0), and after the last a
// token is drawn from p. What matters here is that a draw is an index that a
// rounding near a border would change: sums, exponentials and comparisons
// that decide are in f64. Nearly all of the work is not: a row's maximum is
// exact in any order, its sum of exponentials is taken in f32 first (off by at
// most 5e-6: 2^-22 of each ex2, 2^-23 |x| 2^-x of its argument, one rounding a
// term), and a comparison closer than 1e-4 to its border is decided again
// with the sum in f64. Only the one row a sequence draws from is summed in
// f64 throughout.
//
// A cluster a sequence: its CTAs take the rows between them (one read of each
// from HBM, which bounds the large calls), the verdicts meet in the first
// CTA's shared memory, then all share the drawn row, in slices in order, so
// that the prefix sums over slices, threads and values give the index.

#include <cooperative_groups.h>

#include <cfloat>

#include "kv4_host.h"

namespace nd {

namespace cg = cooperative_groups;

constexpr int VF_THREADS = 512, VF_MAX_DRAFT = 64;
constexpr float LOG2E = 1.4426950408889634f;

struct VerifyArgs {
    long long l_seq, l_row, q_seq, q_row;
    const int32_t* draft;   // [seqs][T]
    const int32_t* counts;  // [seqs] or NULL
    const float* u;         // [seqs][T + 1]
    const float* temp;      // [seqs]
    const float* q;         // or NULL
    int seqs, T, V;
    bool l_vec;
    int32_t *tokens, *accepted;  // [seqs][T + 1], [seqs]
    float* probs;                // [seqs][T + 1]
};

// A row's largest logit, its first place, and sum exp((l - top) / temperature).
struct RowStats {
    float top;
    int at;       // -1: a NaN, or nothing above -infinity
    double sum;
};

__device__ __forceinline__ float vf_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <typename T>
__device__ __forceinline__ double term(const T* row, int j, float top, double inv) {
    return exp(((double)(float)row[j] - (double)top) * inv);
}

__device__ __forceinline__ double block_sum(double x, double* red) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 16; o; o /= 2) x += __shfl_xor_sync(0xffffffffu, x, o);
    __syncthreads();
    if (lane == 0) red[warp] = x;
    __syncthreads();
    double s = 0.0;
    for (int w = 0; w < VF_THREADS / 32; w++) s += red[w];
    return s;
}

// One pass over a row by the CTA; every thread returns the result.
template <typename T>
__device__ RowStats row_stats(const T* row, int V, float scale2, bool vec, double* red, float* redf, int* redi) {
    constexpr int PER = 16 / sizeof(T);
    float top = -INFINITY, sum = 0.f;
    int at = V;
    bool nan = false;
    auto take = [&](const float* x, int n, int j0) {
        float m = top;
#pragma unroll
        for (int i = 0; i < PER; i++)
            if (i < n) {
                nan |= x[i] != x[i];
                if (x[i] > m) m = x[i], at = j0 + i;
            }
        if (m > top) {
            sum *= vf_ex2((top - m) * scale2);  // top = -infinity: sum is 0
            top = m;
        }
        if (top == -INFINITY) return;
#pragma unroll
        for (int i = 0; i < PER; i++)
            if (i < n) sum += vf_ex2((x[i] - top) * scale2);
    };
    if (vec) {
        const int units = V / PER;
        for (int k = threadIdx.x; k < units; k += VF_THREADS) {
            float x[8];
            if constexpr (sizeof(T) == 4) {
                const float4 f = __ldg((const float4*)row + k);
                x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w;
            } else {
                load8(row + 8 * k, true, x);
            }
            take(x, PER, k * PER);
        }
        for (int j = units * PER + threadIdx.x; j < V; j += VF_THREADS) {
            const float x[8] = {(float)row[j]};
            take(x, 1, j);
        }
    } else {
        for (int j = threadIdx.x; j < V; j += VF_THREADS) {
            const float x[8] = {(float)row[j]};
            take(x, 1, j);
        }
    }
    // the block's largest, the first place that has it
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float m = top;
    int place = at;
#pragma unroll
    for (int o = 16; o; o /= 2) {
        const float om = __shfl_xor_sync(0xffffffffu, m, o);
        const int op = __shfl_xor_sync(0xffffffffu, place, o);
        if (om > m || (om == m && op < place)) m = om, place = op;
        nan |= __shfl_xor_sync(0xffffffffu, (int)nan, o) != 0;
    }
    __syncthreads();
    if (lane == 0) redf[warp] = m, redi[warp] = nan ? -1 : place;
    __syncthreads();
    m = redf[0], place = redi[0];
    nan = place < 0;
    for (int w = 1; w < VF_THREADS / 32; w++) {
        nan |= redi[w] < 0;
        if (redf[w] > m || (redf[w] == m && redi[w] < place)) m = redf[w], place = redi[w];
    }
    RowStats r;
    r.top = m;
    r.at = nan || m == -INFINITY ? -1 : place;
    r.sum = block_sum(top == -INFINITY ? 0.0 : (double)sum * (double)vf_ex2((top - m) * scale2), red);
    return r;
}

template <typename T>
__global__ void __launch_bounds__(VF_THREADS) verify_kernel(VerifyArgs a, const T* __restrict__ logits) {
    cg::cluster_group cluster = cg::this_cluster();
    const int C = cluster.num_blocks(), rank = cluster.block_rank(), s = blockIdx.x / C;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    __shared__ double red[VF_THREADS / 32];
    __shared__ float redf[VF_THREADS / 32];
    __shared__ int redi[VF_THREADS / 32];
    // of the first CTA: each row's verdict and statistics, met through the cluster
    __shared__ int ok[VF_MAX_DRAFT + 1];
    __shared__ float tops[VF_MAX_DRAFT + 1], probs[VF_MAX_DRAFT + 1];
    __shared__ int places[VF_MAX_DRAFT + 1];
    __shared__ double part[2];      // this CTA's sum of exponentials, of the residual
    __shared__ int found, last;     // the drawn place (of the first CTA); the last place that could be drawn
    const int T_ = a.T, V = a.V, n = min(max(a.counts ? __ldg(a.counts + s) : T_, 0), T_);
    const float temp = __ldg(a.temp + s);
    const bool greedy = !(temp > 0.f && LOG2E / temp <= FLT_MAX);
    const double inv = greedy ? 1.0 : 1.0 / (double)temp;
    const float scale2 = greedy ? LOG2E : LOG2E / temp;
    const float* u = a.u + (size_t)s * (T_ + 1);
    const T* rows = logits + s * a.l_seq;
    if (tid == 0) found = V, last = -1;
    int* ok0 = cluster.map_shared_rank(ok, 0);
    float *tops0 = cluster.map_shared_rank(tops, 0), *probs0 = cluster.map_shared_rank(probs, 0);
    int* places0 = cluster.map_shared_rank(places, 0);
    cluster.sync();

    for (int i = rank; i <= n; i += C) {
        const T* row = rows + i * a.l_row;
        const RowStats st = row_stats(row, V, scale2, a.l_vec, red, redf, redi);
        bool take = false;
        double p = 0.0;
        if (i < n && st.at >= 0) {
            const int x = __ldg(a.draft + (size_t)s * T_ + i);
            if (x >= 0 && x < V) {
                const double uq = (double)__ldg(u + i) * (a.q ? (double)__ldg(a.q + s * a.q_seq + i * a.q_row + x) : 1.0);
                if (greedy) {
                    p = x == st.at;
                    take = uq < p;
                } else {
                    const double e = term(row, x, st.top, inv);
                    double z = st.sum;
                    if (fabs(uq * z - e) <= 1e-4 * (fabs(uq * z) + e)) {  // every thread sees the same values
                        double mine = 0.0;
                        for (int j = tid; j < V; j += VF_THREADS) mine += term(row, j, st.top, inv);
                        z = block_sum(mine, red);
                    }
                    p = e / z;
                    take = uq < p;
                }
            }
        }
        if (tid == 0) ok0[i] = take, tops0[i] = st.top, places0[i] = st.at, probs0[i] = (float)p;
        __syncthreads();
    }
    cluster.sync();
    int kept = 0;
    while (kept < n && ok0[kept]) kept++;
    const float top = tops0[kept];
    const int place = places0[kept];

    // the drawn row
    int token = -1;
    float prob = 0.f;
    if (place >= 0 && greedy) {
        // p is one at `place`; what q takes from it leaves it the only token
        token = place;
        prob = 1.f;
    } else if (place >= 0) {
        const T* row = rows + kept * a.l_row;
        const float* q = kept < n && a.q ? a.q + s * a.q_seq + kept * a.q_row : nullptr;
        const int gone = kept < n && !a.q ? __ldg(a.draft + (size_t)s * T_ + kept) : -1;
        const int per = (V + C * VF_THREADS - 1) / (C * VF_THREADS);
        const int lo = min((rank * VF_THREADS + tid) * per, V), hi = min(lo + per, V);
        double mine = 0.0;
        for (int j = lo; j < hi; j++) mine += term(row, j, top, inv);
        const double slice = block_sum(mine, red);
        if (tid == 0) part[0] = slice;
        cluster.sync();
        double z = 0.0;
        for (int r = 0; r < C; r++) z += *cluster.map_shared_rank(part, r);
        const double iz = 1.0 / z;
        bool whole = false;  // p itself, where the residual is all zero
        double total, before, own;
        int top_place;
        auto weight = [&](int j) {
            const double p = term(row, j, top, inv) * iz;
            if (whole) return p;
            if (q) {
                const double r = p - (double)__ldg(q + j);
                return r < 0.0 ? 0.0 : r;
            }
            return j == gone ? 0.0 : p;
        };
        while (true) {
            own = 0.0, top_place = -1;
            for (int j = lo; j < hi; j++) {
                const double w = weight(j);
                own += w;
                if (w > 0.0) top_place = j;
            }
            // what lies before this thread's slice, and in all
            double incl = own;
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const double up = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += up;
            }
            before = __shfl_up_sync(0xffffffffu, incl, 1);
            if (lane == 0) before = 0.0;
            __syncthreads();
            if (lane == 31) red[warp] = incl;
            __syncthreads();
            double all = 0.0;
            for (int w = 0; w < VF_THREADS / 32; w++) {
                if (w == warp) before += all;
                all += red[w];
            }
            if (tid == 0) part[1] = all;
            cluster.sync();
            total = 0.0;
            for (int r = 0; r < C; r++) {
                if (r == rank) before += total;
                total += cluster.map_shared_rank(part, r)[1];
            }
            if (total != 0.0 || whole) break;
            whole = true;
            cluster.sync();
        }
        if (total > 0.0) {
            const double target = fmin(fmax((double)__ldg(u + T_), 0.0), 1.0) * total;
            // the first value at which the running sum passes the target; threads
            // just behind it look too, in case a slice's sum and the next one's
            // start differ in the last bit
            if (top_place >= 0 && before <= target * (1.0 + 1e-9) && before + own > target * (1.0 - 1e-9)) {
                double cum = before;
                for (int j = lo; j < hi; j++) {
                    const double w = weight(j);
                    cum += w;
                    if (w > 0.0 && cum > target) {
                        atomicMin(cluster.map_shared_rank(&found, 0), j);
                        break;
                    }
                }
            }
            if (top_place >= 0) atomicMax(&last, top_place);
            cluster.sync();
            token = *cluster.map_shared_rank(&found, 0);
            if (token >= V) {  // u is 1, or the last bits differ at the very end
                token = -1;
                for (int r = 0; r < C; r++) token = max(token, *cluster.map_shared_rank(&last, r));
            }
            if (token >= 0) prob = (float)(term(row, token, top, inv) * iz);
        } else {
            cluster.sync();
        }
    }
    if (rank == 0)
        for (int i = tid; i <= T_; i += VF_THREADS) {
            const size_t o = (size_t)s * (T_ + 1) + i;
            a.tokens[o] = i < kept ? __ldg(a.draft + (size_t)s * T_ + i) : i == kept ? token : -1;
            a.probs[o] = i < kept ? probs[i] : i == kept ? prob : 0.f;
        }
    if (rank == 0 && tid == 0) a.accepted[s] = kept;
    cluster.sync();  // no CTA leaves while others read its shared memory
}

template <typename T>
static void verify_launch(const VerifyArgs& a, const void* logits, int ctas, cudaStream_t st) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)a.seqs * ctas);
    cfg.blockDim = dim3(VF_THREADS);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = ctas, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, verify_kernel<T>, VerifyArgs(a), (const T*)logits);
    if (e != cudaSuccess) throw std::runtime_error(std::string("nd_op_verify: ") + cudaGetErrorString(e));
    add_launches(1);
}

}  // namespace nd

using namespace nd;

extern "C" int nd_op_verify(int device, int type, const void* logits, long long l_seq, long long l_row, const int* draft,
                            const int* counts, const float* u, const float* temperature, const float* q, long long q_seq,
                            long long q_row, int seqs, int T, int V, int* tokens, int* accepted, float* probs, void* stream) {
    return op_call([&] {
        const char* what = "nd_op_verify";
        auto fail = [&](const std::string& m) { throw std::runtime_error(std::string(what) + ": " + m); };
        if (type != ND_F32 && type != ND_F16 && type != ND_BF16) fail("unknown type");
        if (seqs < 1 || seqs > 1 << 20 || T < 0 || T > VF_MAX_DRAFT || V < 1) fail("needs 1 to 2^20 sequences, 0 to 64 drafted tokens, V >= 1");
        if (!logits || !u || !temperature || !tokens || !accepted || !probs || (T && !draft)) fail("null pointer");
        const int e = type == ND_F32 ? 4 : 2;
        if ((uintptr_t)logits % e || (uintptr_t)q % 4) fail("logits and q must be aligned to their types");
        if (l_seq < 0 || l_row < 0 || q_seq < 0 || q_row < 0) fail("negative strides");
        VerifyArgs a{};
        a.l_seq = l_seq, a.l_row = l_row, a.q_seq = q_seq, a.q_row = q_row;
        a.draft = draft, a.counts = counts, a.u = u, a.temp = temperature, a.q = T ? q : nullptr;
        a.seqs = seqs, a.T = T, a.V = V;
        a.l_vec = (uintptr_t)logits % 16 == 0 && l_seq * e % 16 == 0 && l_row * e % 16 == 0;
        a.tokens = tokens, a.accepted = accepted, a.probs = probs;
        OnDevice on(device, what);
        // a CTA a row up to eight; more where there are few sequences, to share the drawn row
        int ctas = 1;
        while (ctas < 8 && (ctas < T + 1 || seqs * 2 * ctas <= device_sm_count())) ctas *= 2;
        cudaStream_t st = (cudaStream_t)stream;
        if (type == ND_F32) verify_launch<float>(a, logits, ctas, st);
        else if (type == ND_F16) verify_launch<__half>(a, logits, ctas, st);
        else verify_launch<__nv_bfloat16>(a, logits, ctas, st);
    });
}
