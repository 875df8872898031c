// balance.cu -- the router's balance loss: pairs per expert, mean probability per expert, the loss of each sequence and its gradient.
//
// Math, per sequence of L rows (tokens) of E logits, of which the mask leaves n:
//   p = softmax(l), or sigmoid(l_e) / sum of the sigmoids, which is the softmax of log sigmoid(l)
//   f_e = number of ids equal to e,  P_e = sum of p_te,   loss = coef * E / (k n^2) * sum_e f_e P_e      (even load: coef)
//   d l_te = d_loss * coef * E / (k n^2) * p_te * (f_e - sum_j f_j p_tj)  [ * (1 - sigmoid(l_te)) ]
// The counts need the ids alone, which are a few percent of the bytes; with them known one pass over the logits gives both the sums
// and the gradient, so every logit is read once and every gradient written once.  Bound: memory in large batches (16 sequences
// of 8192 x 256 f32 with gradient: 48 us behind 6.5 of counting, 5.6 TB/s), launches and latency in small ones (24 tokens: 4.1 us; 4 x 1000 x 128: 13).
//   balance_kernel a piece of a sequence per CTA, a row by 8, 16 or 32 lanes; sums of a lane in fp32 (of up to 256 values, then in fp64), of the warps and pieces in
//                  fp64 and always in the same order.  Short sequences, and many of them: the pieces of a sequence are a cluster of up to eight CTAs, which count its pairs and add up its sums over
//                  shared memory, one launch in all.  A few long sequences: dozens of pieces each, whose sums the CTAs that finish last add up, behind
//   count_kernel   pairs per expert of a piece of a sequence.
// In the gradient f_e is replaced by f_e - (sum_j f_j) / E, a constant less: it drops out (the p of a row add up to 1), and the difference
// that remains does not lose the digits of the load all experts share.
#include <cuda_bf16.h>

#include <type_traits>

#include "common.cuh"
#include "kernels.h"

namespace chimere {
namespace {

constexpr int kB_Threads = 256, kB_Warps = kB_Threads / 32;
constexpr int kB_CtasPerSm = 3;
constexpr int kB_Turns = 16, kB_LongTurns = 64;   // of a warp, between two sums in fp64; from more turns than these on
constexpr int kB_Group = 32;          // pieces that are added up together, and groups of them
constexpr int kB_CountCluster = 8, kB_MaxCountPieces = 16;
constexpr int kB_CountIds = 4096;     // ids of a counting CTA, where that gives few enough of them

struct BalanceParams {
    const void* logits;
    int64_t ld, stride_s;
    const int32_t* ids;               // null: the counts are given (backward)
    const uint8_t* mask;              // or null
    int S, L, E, k, mode;
    float coef;
    float* loss;                      // null: backward
    int32_t* counts;
    float* prob;
    int32_t* tokens;
    const float* d_loss;              // or null = 1
    void* d_logits;                   // or null
    int64_t ldd, stride_ds;
    int vec;                          // rows of logits and gradient can be read and written four values at a time
    int pieces, rows;                 // of a sequence (count_pieces = 0: the CTAs of a cluster); rows of a piece
    int count_pieces, count_rows;     // of a sequence, by a cluster each (0: counted here); rows of a CTA
    int32_t* count_part;              // [S][count_pieces][E + 1]
    float* part;                      // [S][pieces][E]
    double* group_part;               // [S][groups][E]
    int32_t* counters;                // [S][groups + 1]
};
__host__ __device__ inline int groups_of(int pieces) { return (pieces + kB_Group - 1) / kB_Group; }

__device__ __forceinline__ bool counted(const BalanceParams& p, int64_t row) { return !p.mask || p.mask[row] != 0; }

// Pairs and tokens of rows [r0, r1) of sequence s, added to hist[E] and hist[E + 1] (shared memory).
__device__ __forceinline__ void count_rows(const BalanceParams& p, int s, int r0, int r1, int* hist) {
    const int64_t base = (int64_t)s * p.L;
    const int32_t* ids = p.ids + (base + r0) * p.k;
    auto add = [&](int e) { if ((uint32_t)e < (uint32_t)p.E) atomicAdd(hist + e, 1); };
    if (!p.mask) {
        if (threadIdx.x == 0) atomicAdd(hist + p.E, r1 - r0);
        const int total = (r1 - r0) * p.k, head = min(total, (int)(-((uintptr_t)ids >> 2) & 3)), quads = (total - head) >> 2;   // (16-byte boundaries)
        const int4* ids4 = reinterpret_cast<const int4*>(ids + head);
#pragma unroll 4
        for (int i = threadIdx.x; i < quads; i += kB_Threads) {
            const int4 v = __ldg(ids4 + i);
            add(v.x); add(v.y); add(v.z); add(v.w);
        }
        const int rest = total - 4 * quads;   // in front and behind
        if ((int)threadIdx.x < rest) add(ids[(int)threadIdx.x < head ? threadIdx.x : threadIdx.x + 4 * quads]);
    } else {
        int mine = 0;
        const int rows = r1 - r0, per = kB_Threads / min(p.k, 8), sub = threadIdx.x / per;   // up to eight threads per row, neighbours on neighbouring rows
#pragma unroll 2
        for (int r = threadIdx.x % per; r < rows && sub < min(p.k, 8); r += per) {
            const bool on = p.mask[base + r0 + r] != 0;
            mine += on && sub == 0;
            for (int j = sub; j < p.k; j += 8) {
                const int e = __ldg(ids + (int64_t)r * p.k + j);   // (on its way together with the mask)
                if (on) add(e);
            }
        }
        mine = __reduce_add_sync(0xffffffffu, mine);
        if ((threadIdx.x & 31) == 0 && mine) atomicAdd(hist + p.E, mine);
    }
}

__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ int ld_peer(const int* mine, int rank) {   // the value at this place in another CTA of the cluster
    uint32_t a;
    int v;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(mine)), "r"(rank));
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}

// A cluster of eight CTAs counts a piece of a sequence; its counts meet in shared memory.
__global__ void __cluster_dims__(kB_CountCluster, 1, 1) __launch_bounds__(kB_Threads) count_kernel(BalanceParams p) {
    __shared__ int hist[kMaxExperts + 1];
    griddep_launch();
    const int rank = blockIdx.x % kB_CountCluster, s = blockIdx.x / kB_CountCluster / p.count_pieces, c = blockIdx.x / kB_CountCluster % p.count_pieces;
    for (int e = threadIdx.x; e <= p.E; e += kB_Threads) hist[e] = 0;
    if (c == 0 && rank == 0) {
        const int n = groups_of(p.pieces) + 1;
        for (int i = threadIdx.x; i < n; i += kB_Threads) p.counters[(int64_t)s * n + i] = 0;
    }
    __syncthreads();
    const int64_t at = ((int64_t)c * kB_CountCluster + rank) * p.count_rows;
    const int r0 = (int)min(at, (int64_t)p.L), r1 = (int)min(at + p.count_rows, (int64_t)p.L);
    count_rows(p, s, r0, r1, hist);
    cluster_barrier();
    int32_t* out = p.count_part + ((int64_t)s * p.count_pieces + c) * (p.E + 1);
    for (int e = (int)threadIdx.x * kB_CountCluster + rank; e <= p.E; e += kB_CountCluster * kB_Threads) {
        int n = 0;
#pragma unroll
        for (int i = 0; i < kB_CountCluster; ++i) n += ld_peer(hist + e, i);
        out[e] = n;
    }
    cluster_barrier();   // (a CTA's counts stay until all have read them)
}

template <int TYPE> __device__ __forceinline__ float to_float(uint32_t bits) { return TYPE == CHIMERE_TYPE_F16 ? h2f(bits) : __uint_as_float(bits << 16); }
// Four neighbouring logits as they lie in memory; those that are not there are -infinity.  n: values there are (FULL: 0 or 4, else 0 .. 4).
template <int TYPE> struct Four {
    static constexpr int kWords = TYPE == CHIMERE_TYPE_F32 ? 4 : 2;
    static constexpr uint32_t kNone = TYPE == CHIMERE_TYPE_F32 ? 0xFF800000u : TYPE == CHIMERE_TYPE_F16 ? 0xFC00FC00u : 0xFF80FF80u;
    uint32_t w[kWords];
    template <bool FULL>
    __device__ __forceinline__ void load(const void* base, int64_t at, int n, bool vec) {
        const uint32_t* q = reinterpret_cast<const uint32_t*>(reinterpret_cast<const char*>(base) + at * kWords);
        if (FULL || (vec && n == 4)) {
#pragma unroll
            for (int i = 0; i < kWords; ++i) w[i] = kNone;
            if (n) {
                if constexpr (TYPE == CHIMERE_TYPE_F32) {
                    const uint4 a = __ldcs(reinterpret_cast<const uint4*>(q));
                    w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
                } else {
                    const uint2 a = __ldcs(reinterpret_cast<const uint2*>(q));
                    w[0] = a.x; w[1] = a.y;
                }
            }
        } else if constexpr (TYPE == CHIMERE_TYPE_F32) {
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = i < n ? q[i] : kNone;
        } else {
            const uint16_t* h = reinterpret_cast<const uint16_t*>(q);
#pragma unroll
            for (int i = 0; i < 2; ++i) w[i] = (2 * i < n ? h[2 * i] : kNone & 0xFFFFu) | ((2 * i + 1 < n ? h[2 * i + 1] : kNone & 0xFFFFu) << 16);
        }
    }
    __device__ __forceinline__ float value(int i) const {
        if constexpr (TYPE == CHIMERE_TYPE_F32) return __uint_as_float(w[i]);
        else if (TYPE == CHIMERE_TYPE_BF16 && (i & 1)) return __uint_as_float(w[i / 2] & 0xFFFF0000u);
        else return to_float<TYPE>((w[i / 2] >> (16 * (i & 1))) & 0xFFFFu);
    }
};
template <int TYPE> __device__ __forceinline__ uint32_t two(float a, float b) {
    if (TYPE == CHIMERE_TYPE_F16) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <int TYPE, bool FULL>
__device__ __forceinline__ void store4(void* base, int64_t at, int n, bool vec, const float (&v)[4]) {
    if constexpr (TYPE == CHIMERE_TYPE_F32) {
        float* q = reinterpret_cast<float*>(base) + at;
        if (FULL || (vec && n == 4)) {
            if (n) __stcs(reinterpret_cast<float4*>(q), make_float4(v[0], v[1], v[2], v[3]));
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) if (i < n) q[i] = v[i];
        }
    } else {
        uint16_t* q = reinterpret_cast<uint16_t*>(base) + at;
        const uint2 w = make_uint2(two<TYPE>(v[0], v[1]), two<TYPE>(v[2], v[3]));
        if (FULL || (vec && n == 4)) {
            if (n) __stcs(reinterpret_cast<uint2*>(q), w);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) if (i < n) q[i] = (uint16_t)((i < 2 ? w.x : w.y) >> (16 * (i & 1)));
        }
    }
}
// over the LANES lanes of a row, several rows at a time
template <int LANES, int N> __device__ __forceinline__ void lanes_max(float (&v)[N]) {
    if constexpr (LANES == 32) {
#pragma unroll
        for (int u = 0; u < N; ++u) asm volatile("redux.sync.max.f32 %0, %0, 0xffffffff;" : "+f"(v[u]));   // (passes over NaNs, as fmaxf does)
    } else {
#pragma unroll
        for (int d = LANES / 2; d > 0; d >>= 1)
#pragma unroll
            for (int u = 0; u < N; ++u) v[u] = fmaxf(v[u], __shfl_xor_sync(0xffffffffu, v[u], d));
    }
}
template <int LANES, int N> __device__ __forceinline__ void lanes_sum(float (&v)[N]) {
#pragma unroll
    for (int d = LANES / 2; d > 0; d >>= 1) {
        float o[N];
#pragma unroll
        for (int u = 0; u < N; ++u) o[u] = __shfl_xor_sync(0xffffffffu, v[u], d);
#pragma unroll
        for (int u = 0; u < N; ++u) v[u] += o[u];
    }
}
__device__ __forceinline__ float rcp(float v) {   // (off by one step at most)
    float r;
    asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

// exp of two values that are not positive: 2^h times 1 + r with h = x log2(e) rounded and r = x - h ln(2) what the rounding left out (ln(2) in two
// parts).  Below -150 it is 0 (a NaN stays one); off by the two steps of ex2 and half a step of the last product.
__device__ __forceinline__ uint64_t exp_pair(uint64_t x) {
    float a, b;
    unpack2(x, a, b);
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(-150.0f));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(b) : "f"(-150.0f));
    x = pack2f(a, b);
    const uint64_t h = mul2(x, pack2f(1.44269504f, 1.44269504f));
    uint64_t r = fma2(h, pack2f(-0.693147182f, -0.693147182f), x);
    r = fma2(h, pack2f(1.90465421e-9f, 1.90465421e-9f), r);
    unpack2(h, a, b);
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(a));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(b));
    const uint64_t e = pack2f(a, b);
    return fma2(e, r, e);
}

template <class Part> struct BalanceShared {
    int hist[kMaxExperts + 1];        // of the whole sequence; [E]: tokens
    int mine[kMaxExperts + 1];        // of this CTA's rows (cluster)
    float sums[kMaxExperts];          // ... and their probabilities
    float g[kMaxExperts];
    Part part[kB_Warps][kMaxExperts];
    double sum[kB_Warps];
    int last;
};

// prob and loss from the probabilities' sums: sum_of(e), thread e % kB_Threads asks
template <class Shared, class Sum>
__device__ __forceinline__ void finish_sequence(const BalanceParams& p, Shared& sh, int s, Sum sum_of) {
    const int n = sh.hist[p.E], tid = threadIdx.x;
    double dot = 0.0;
    for (int e = tid; e < p.E; e += kB_Threads) {
        const double P = sum_of(e);
        dot += (double)sh.hist[e] * P;
        p.prob[(int64_t)s * p.E + e] = n > 0 ? (float)(P / n) : 0.0f;
        p.counts[(int64_t)s * p.E + e] = sh.hist[e];
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
    if ((tid & 31) == 0) sh.sum[tid >> 5] = dot;
    __syncthreads();
    if (tid == 0) {
        dot = 0.0;
        for (int w = 0; w < kB_Warps; ++w) dot += sh.sum[w];
        p.loss[s] = n > 0 ? (float)((double)p.coef * p.E / ((double)p.k * n * n) * dot) : 0.0f;
        p.tokens[s] = n;
    }
}

// A row by LANES lanes, G groups of four values each: lane i owns values 4 (i + LANES g) .. + 3.
// FULL: as many logits as the lanes hold, rows that are read and written four values at a time: no lane looks at what it has.
// LONG: pieces of more than kB_LongTurns turns of a warp.  A lane adds up a probability per row of its own, off by their number in half-steps of fp32 at most (mean
// probabilities of 2^23 equal rows were 437 off), so there the sums of kB_Turns turns are added up in fp64.  us, without / with them: 60 x 9001 x 256 bf16, gradient 195 / 190, f32 269 / 275;
// 57 x 70003 x 31 f32 318 / 359, bf16 549 / 545.  A kernel of its own: in the other one these sums cost 0.4 us of 4 in small calls and up to a quarter in spilled registers (8 x
// 8192 x 255 bf16 sigmoid 37.5, 48.6 with a loop around the turns).
template <int G> __host__ __device__ constexpr int rows_at_a_time() { return G == 2 ? 2 : 4; }
template <int LANES, int G> __host__ __device__ constexpr int turn_rows() { return kB_Warps * (32 / LANES) * rows_at_a_time<G>(); }
template <int TYPE, int LANES, int G, bool SIGMOID, bool FULL, bool LONG>
__global__ void __launch_bounds__(kB_Threads, kB_CtasPerSm) balance_kernel(BalanceParams p) {
    constexpr int kRows = 32 / LANES, kU = rows_at_a_time<G>(), kStep = turn_rows<LANES, G>();   // rows of a warp at a time: kRows * kU
    __shared__ BalanceShared<typename std::conditional<LONG, double, float>::type> sh;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, sub = lane / LANES, i4 = 4 * (lane % LANES);
    const int s = blockIdx.x / p.pieces, piece = blockIdx.x % p.pieces;
    const int r0 = (int)min((int64_t)piece * p.rows, (int64_t)p.L), r1 = (int)min((int64_t)r0 + p.rows, (int64_t)p.L);
    const bool stats = p.loss != nullptr, grad = p.d_logits != nullptr;

    // this warp's first rows
    const int row_first = r0 + warp * (kRows * kU);
    int there[G];
#pragma unroll
    for (int j = 0; j < G; ++j) there[j] = FULL ? 4 : max(0, min(4, p.E - (i4 + 4 * LANES * j)));
    Four<TYPE> next[kU][G];
    // (a row that is not there, or that the mask leaves out, is one of -infinities: no probabilities, no gradient)
    auto fetch = [&](int row0) {
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            const int r = row0 + u * kRows + sub;
            const bool on = r < r1 && counted(p, (int64_t)s * p.L + r);
            const int64_t at = (int64_t)s * p.stride_s + (int64_t)r * p.ld + i4;
#pragma unroll
            for (int j = 0; j < G; ++j) next[u][j].template load<FULL>(p.logits, at + 4 * LANES * j, on ? there[j] : 0, p.vec);
        }
    };
    fetch(row_first);

    // the pairs of the whole sequence
    if (!p.ids) {
        for (int e = tid; e < p.E; e += kB_Threads) sh.hist[e] = p.counts[(int64_t)s * p.E + e];
        if (tid == 0) sh.hist[p.E] = p.tokens[s];
    } else if (p.count_pieces == 0) {
        int* mine = p.pieces == 1 ? sh.hist : sh.mine;
        for (int e = tid; e <= p.E; e += kB_Threads) mine[e] = 0;
        __syncthreads();
        count_rows(p, s, r0, r1, mine);
        if (p.pieces > 1) {
            cluster_barrier();
            for (int e = tid; e <= p.E; e += kB_Threads) {
                int n = 0;
                for (int i = 0; i < p.pieces; ++i) n += ld_peer(sh.mine + e, i);
                sh.hist[e] = n;
            }
        }
    } else {
        griddep_wait();
        const int32_t* part = p.count_part + (int64_t)s * p.count_pieces * (p.E + 1);
        for (int e = tid; e <= p.E; e += kB_Threads) {
            int c = 0;
#pragma unroll 4
            for (int i = 0; i < p.count_pieces; ++i) c += __ldcg(part + (int64_t)i * (p.E + 1) + e);
            sh.hist[e] = c;
        }
    }
    __syncthreads();
    if (grad) {
        int low = 0, high = 0;   // (the counts of several ranks may add up to more than 31 bits)
        for (int e = lane; e < p.E; e += 32) { low += sh.hist[e] & 0xFFFF; high += sh.hist[e] >> 16; }
        const double all = (double)__reduce_add_sync(0xffffffffu, high) * 65536.0 + __reduce_add_sync(0xffffffffu, low);
        const double n = sh.hist[p.E], c = n > 0 ? (double)p.coef * p.E / (p.k * n * n) * (p.d_loss ? (double)p.d_loss[s] : 1.0) : 0.0;
        for (int e = tid; e < p.E; e += kB_Threads) sh.g[e] = (float)(c * (sh.hist[e] - all / p.E));
        __syncthreads();
    }
    uint64_t g[G][2], acc[G][2];
#pragma unroll
    for (int j = 0; j < G; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int e = i4 + 4 * LANES * j + 2 * i;
            acc[j][i] = 0;
            g[j][i] = pack2f(grad && e < p.E ? sh.g[e] : 0.0f, grad && e + 1 < p.E ? sh.g[e + 1] : 0.0f);
        }

    if (LONG) {
        for (int e = lane; e < p.E; e += 32) sh.part[warp][e] = 0;
        __syncwarp();
    }
    auto fold = [&]() {   // the sums of these turns over the rows of a warp
        int t = tid;
        if (LONG) asm volatile("mov.u32 %0, %%tid.x;" : "=r"(t));   // (asked for again, so that no place of these sums is kept in registers through the turns)
        const int w = t >> 5, mine = (t & 31) / LANES, first = 4 * ((t & 31) % LANES);
#pragma unroll
        for (int j = 0; j < G; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float a, b;
                unpack2(acc[j][i / 2], a, b);
                float v = i & 1 ? b : a;
#pragma unroll
                for (int d = LANES; d < 32; d <<= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
                const int e = first + 4 * LANES * j + i;
                if (mine == 0 && e < p.E) {
                    if (LONG) sh.part[w][e] += v;
                    else sh.part[w][e] = v;
                }
            }
    };
    int turns = 0;
#pragma unroll 1
    for (int row0 = row_first; row0 < r1; row0 += kStep) {
        if (LONG && turns++ == kB_Turns) {
            fold();
#pragma unroll
            for (int j = 0; j < G; ++j) acc[j][0] = acc[j][1] = 0;
            turns = 1;
        }
        uint64_t v[kU][G][2];   // two values each
        // step by step for all of the warp's rows, so that one row's exchanges between lanes pass behind the others'
        float mx[kU], sum[kU], dot[kU];
        uint64_t slope[SIGMOID ? kU : 1][G][2];   // 1 - sigmoid(l)
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            mx[u] = next[u][0].value(0);
#pragma unroll
            for (int j = 0; j < G; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) mx[u] = fmaxf(mx[u], next[u][j].value(i));
        }
        lanes_max<LANES>(mx);
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            if (mx[u] == __uint_as_float(0xFF800000u)) mx[u] = 0.0f;   // (-infinities stay zeros, a NaN among them stays one)
            // l becomes its part of the sum: exp(l - max), or sigmoid(l) -- in rows whose sigmoids are all below 1e-26, where they are exp(l) to
            // fp32's last digit and could leave its range, the same exp(l - max)
            const bool low = SIGMOID && mx[u] < -60.0f;
            const float shift = !SIGMOID || low ? -mx[u] : 0.0f, one = low ? 0.0f : 1.0f;
            const uint64_t shift2 = pack2f(shift, shift), one2 = pack2f(one, one);
            uint64_t sum2 = 0, dot2 = 0;
#pragma unroll
            for (int j = 0; j < G; ++j)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float a = next[u][j].value(2 * i), b = next[u][j].value(2 * i + 1);
                    uint64_t& l = v[u][j][i];
                    if (SIGMOID) {
                        const uint64_t t = exp_pair(add2(pack2f(-fabsf(a), -fabsf(b)), shift2));
                        float d0, d1;
                        unpack2(fma2(t, one2, pack2f(1.0f, 1.0f)), d0, d1);
                        const uint64_t q = pack2f(rcp(d0), rcp(d1));
                        float q0, q1, t0, t1;
                        unpack2(q, q0, q1);
                        unpack2(mul2(t, q), t0, t1);
                        const bool up0 = a >= 0.0f, up1 = b >= 0.0f;
                        slope[u][j][i] = pack2f(up0 ? t0 : q0, up1 ? t1 : q1);
                        l = pack2f(up0 ? q0 : t0, up1 ? q1 : t1);
                    } else {
                        l = exp_pair(add2(pack2f(a, b), shift2));
                    }
                    sum2 = add2(sum2, l);
                    dot2 = fma2(l, g[j][i], dot2);
                }
            float a, b;
            unpack2(sum2, a, b);
            sum[u] = a + b;
            unpack2(dot2, a, b);
            dot[u] = a + b;
        }
        fetch(row0 + kStep);   // (the rows after these are on their way while these are finished, and copied nowhere)
        lanes_sum<LANES>(sum);
        if (grad) lanes_sum<LANES>(dot);
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            const float inv = sum[u] == 0.0f ? 0.0f : __frcp_rn(sum[u]);
            const uint64_t inv2 = pack2f(inv, inv);
            dot[u] *= inv;
#pragma unroll
            for (int j = 0; j < G; ++j)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    v[u][j][i] = mul2(v[u][j][i], inv2);
                    acc[j][i] = add2(acc[j][i], v[u][j][i]);
                }
        }
        if (!grad) continue;
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            const int r = row0 + u * kRows + sub;
            const int64_t at = (int64_t)s * p.stride_ds + (int64_t)r * p.ldd + i4;
            const uint64_t less = pack2f(-dot[u], -dot[u]);
#pragma unroll
            for (int j = 0; j < G; ++j) {
                float d[4];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    uint64_t w = mul2(v[u][j][i], add2(g[j][i], less));
                    if (SIGMOID) w = mul2(w, slope[u][j][i]);
                    unpack2(sum[u] == 0.0f ? 0 : w, d[2 * i], d[2 * i + 1]);   // (zero also where grad_loss is not finite)
                }
                store4<TYPE, FULL>(p.d_logits, at + 4 * LANES * j, r < r1 ? there[j] : 0, p.vec, d);
            }
        }
    }
    griddep_launch();
    if (!stats) return;
    fold();

    // the piece's sums
    __syncthreads();
    auto of_piece = [&](int e) {
        double v = 0.0;
#pragma unroll
        for (int w = 0; w < kB_Warps; ++w) v += (double)sh.part[w][e];
        return v;
    };
    if (p.count_pieces == 0) {
        if (p.pieces > 1) {
            for (int e = tid; e < p.E; e += kB_Threads) sh.sums[e] = (float)of_piece(e);
            cluster_barrier();
            if (piece == 0) finish_sequence(p, sh, s, [&](int e) {
                double v = 0.0;
                for (int i = 0; i < p.pieces; ++i) v += (double)__int_as_float(ld_peer(reinterpret_cast<int*>(sh.sums) + e, i));
                return v;
            });
            cluster_barrier();   // (a CTA's sums stay until they have been read)
        } else {
            finish_sequence(p, sh, s, of_piece);
        }
        return;
    }
    const int groups = groups_of(p.pieces), group = piece / kB_Group, in_group = min(kB_Group, p.pieces - group * kB_Group);
    float* part = p.part + (int64_t)s * p.pieces * p.E;
    for (int e = tid; e < p.E; e += kB_Threads) __stcg(part + (int64_t)piece * p.E + e, (float)of_piece(e));
    __syncthreads();
    if (tid == 0) sh.last = atom_add_acq_rel_gpu(p.counters + (int64_t)s * (groups + 1) + group, 1) == in_group - 1;
    __syncthreads();
    if (!sh.last) return;
    auto of_group = [&](int e) {
        double v = 0.0;
#pragma unroll 8
        for (int i = 0; i < in_group; ++i) v += (double)__ldcg(part + (int64_t)(group * kB_Group + i) * p.E + e);
        return v;
    };
    if (groups == 1) {
        finish_sequence(p, sh, s, of_group);
        return;
    }
    double* gpart = p.group_part + (int64_t)s * groups * p.E;
    for (int e = tid; e < p.E; e += kB_Threads) __stcg(gpart + (int64_t)group * p.E + e, of_group(e));
    __syncthreads();
    if (tid == 0) sh.last = atom_add_acq_rel_gpu(p.counters + (int64_t)s * (groups + 1) + groups, 1) == groups - 1;
    __syncthreads();
    if (!sh.last) return;
    finish_sequence(p, sh, s, [&](int e) {
        double v = 0.0;
#pragma unroll 8
        for (int i = 0; i < groups; ++i) v += __ldcg(gpart + (int64_t)i * p.E + e);
        return v;
    });
}

template <int TYPE, bool SIGMOID>
cudaError_t launch_balance_type(const BalanceParams& p, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((int64_t)p.S * p.pieces));
    cfg.blockDim = dim3(kB_Threads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    cfg.attrs = attr;
    if (p.count_pieces) {
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.numAttrs = 1;
    } else if (p.pieces > 1 && p.ids) {
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = (unsigned)p.pieces;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.numAttrs = 1;
    }
    auto go = [&](auto lanes, auto groups) {
        constexpr int LANES = decltype(lanes)::value, G = decltype(groups)::value;
        const bool full = p.vec && p.E == 4 * LANES * G, many = p.loss && p.rows > kB_LongTurns * turn_rows<LANES, G>();
        auto kernel = many ? full ? balance_kernel<TYPE, LANES, G, SIGMOID, true, true> : balance_kernel<TYPE, LANES, G, SIGMOID, false, true>
                           : full ? balance_kernel<TYPE, LANES, G, SIGMOID, true, false> : balance_kernel<TYPE, LANES, G, SIGMOID, false, false>;
        return cudaLaunchKernelEx(&cfg, kernel, p);
    };
    using std::integral_constant;
    if (p.E <= 32) return go(integral_constant<int, 8>(), integral_constant<int, 1>());
    if (p.E <= 64) return go(integral_constant<int, 16>(), integral_constant<int, 1>());
    if (p.E <= 128) return go(integral_constant<int, 32>(), integral_constant<int, 1>());
    return go(integral_constant<int, 32>(), integral_constant<int, 2>());
}
template <int TYPE> cudaError_t launch_balance_mode(const BalanceParams& p, cudaStream_t stream) {
    return p.mode == CHIMERE_ROUTE_SIGMOID_NORM_SCALE ? launch_balance_type<TYPE, true>(p, stream) : launch_balance_type<TYPE, false>(p, stream);
}
cudaError_t launch_balance(const BalanceParams& p, int type, cudaStream_t stream) {
    return type == CHIMERE_TYPE_F32 ? launch_balance_mode<CHIMERE_TYPE_F32>(p, stream)
         : type == CHIMERE_TYPE_F16 ? launch_balance_mode<CHIMERE_TYPE_F16>(p, stream) : launch_balance_mode<CHIMERE_TYPE_BF16>(p, stream);
}

// Pieces of a sequence.  With the counting in front: as many CTAs as run at once.  In clusters: up to eight, at least kB_PieceRows rows in each; taken
// for short sequences, and for so many of them that eight pieces of each fill the GPU.
// us, with gradient, in clusters / with counting in front, of 1, 4, 16 and 32 sequences: 256 f32 logits, 512 rows 9.7 / 10.0, 10.2 / 10.0, 11.8 / 12.9, 12.4 / 15.4; 1024 rows
// 13.7 / 11.0, 14.1 / 12.0, 17.1 / 15.4, 17.6 / 20.0; 2048 rows 21.9 / 12.8, 21.8 / 14.0, 27.5 / 20.2, 29.0 / 29.5.  128 bf16 logits, sigmoid, 512 rows 8.0 / 8.7, 8.6 / 9.0,
// 10.1 / 10.6, 10.4 / 14.0; 1024 rows 11.0 / 9.4, 11.4 / 10.2, 14.3 / 13.9, 14.8 / 17.5; 2048 rows 16.7 / 11.0, 17.4 / 12.3, 22.8 / 17.7, 23.3 / 25.0.  (Between 512 and 1024
// rows clusters are up to 3 us slower for few sequences, up to 3 faster for many.)
constexpr int kB_PieceRows = 32, kB_Cluster = 8, kB_ClusterRows = 1024, kB_Sms = 148;   // (the scratch's size goes by these: constants)
struct Plan { int pieces, rows, count_pieces, count_rows; };
Plan plan_of(int64_t S, int L, int k) {
    Plan r{};
    constexpr int64_t slots = kB_CtasPerSm * kB_Sms;
    if (L <= kB_ClusterRows || S * kB_Cluster >= slots) {
        // waves times rows, a CTA's fixed cost taken for those of kB_PieceRows
        int64_t best = 0;
        for (int n = 1; n <= kB_Cluster && (n == 1 || (int64_t)(n - 1) * kB_PieceRows < L); ++n) {
            const int64_t cost = ((S * n + slots - 1) / slots) * (((int64_t)L + n - 1) / n + kB_PieceRows);
            if (n == 1 || cost < best) { best = cost; r.pieces = n; }
        }
        r.rows = (int)(((int64_t)L + r.pieces - 1) / r.pieces);
        return r;
    }
    const int64_t n = slots / S;      // (rounded down: one more wave for a few pieces would double the time)
    r.rows = (int)((L + n - 1) / n);
    r.rows = r.rows < kB_PieceRows ? kB_PieceRows : r.rows;
    r.pieces = (int)(((int64_t)L + r.rows - 1) / r.rows);
    int64_t c = ((int64_t)L * k + kB_CountCluster * kB_CountIds - 1) / (kB_CountCluster * kB_CountIds);
    c = c > kB_MaxCountPieces ? kB_MaxCountPieces : c;
    r.count_pieces = (int)c;
    r.count_rows = (int)((L + c * kB_CountCluster - 1) / (c * kB_CountCluster));
    return r;
}
static_assert(kB_CtasPerSm * kB_Sms <= kB_Group * kB_Group, "two levels of sums");
inline size_t up256(size_t v) { return (v + 255) & ~(size_t)255; }
struct Scratch { size_t count_part, part, group_part, counters, total; };
Scratch scratch_of(const Plan& r, int64_t S, int E) {
    Scratch a{};
    if (r.count_pieces == 0) return a;
    size_t o = 0;
    a.group_part = o; o += up256((size_t)S * groups_of(r.pieces) * E * 8);
    a.part = o; o += up256((size_t)S * r.pieces * E * 4);
    a.count_part = o; o += up256((size_t)S * r.count_pieces * (E + 1) * 4);
    a.counters = o; o += up256((size_t)S * (groups_of(r.pieces) + 1) * 4);
    a.total = o;
    return a;
}
inline bool misaligned(const void* p, int to) { return ((uintptr_t)p & (uintptr_t)(to - 1)) != 0; }
inline int rc_of(cudaError_t e) { return e == cudaSuccess ? 0 : -(100 + (int)e); }

int check_dims(int64_t S, int64_t L, int E, int k, int mode, int type, int64_t ld, int64_t stride_s) {
    if (S < 0 || L < 0 || S > 0x7FFFFFFF / 1024 || L > 0x7FFFFF00 || E <= 0 || E > kMaxExperts || k <= 0 || k > kMaxExperts) return -2;
    if (L > 0 && S > 0x7FFFFFFF / L) return -2;      // (counts and token numbers are 32-bit)
    if (L > 0 && k > 0x7FFFFFFF / L) return -2;
    if (mode != CHIMERE_ROUTE_SOFTMAX_RENORM && mode != CHIMERE_ROUTE_SIGMOID_NORM_SCALE) return -2;
    if (ld < E || (S > 1 && stride_s < 0)) return -2;
    if (type != CHIMERE_TYPE_F32 && type != CHIMERE_TYPE_F16 && type != CHIMERE_TYPE_BF16) return -3;
    return 0;
}
int vectors(const void* p, int64_t ld, int64_t stride, int E, int type) {
    const int size = type == CHIMERE_TYPE_F32 ? 4 : 2;
    return E % 4 == 0 && !misaligned(p, 4 * size) && ld % 4 == 0 && stride % 4 == 0;
}

}  // namespace
}  // namespace chimere

using namespace chimere;

extern "C" {

int64_t chimere_b200_balance_loss_bytes(int64_t S, int64_t L, int E, int top_k) {
    const int rc = check_dims(S, L, E, top_k, CHIMERE_ROUTE_SOFTMAX_RENORM, CHIMERE_TYPE_F32, E, 0);
    return rc ? rc : S == 0 ? 0 : (int64_t)scratch_of(plan_of(S, (int)L, top_k), S, E).total;
}

int chimere_b200_balance_loss(const void* d_logits, int type, int64_t ld, int64_t stride_s, const int32_t* d_topk_idx, const uint8_t* d_mask, int64_t S, int64_t L, int E,
                              int top_k, int route_mode, float coef, float* d_loss, int32_t* d_counts, float* d_prob, int32_t* d_tokens,
                              const float* d_grad_loss, void* d_grad_logits, int64_t ld_grad, int64_t stride_grad_s, void* d_ws, size_t ws_bytes, cudaStream_t stream) {
    const int rc = check_dims(S, L, E, top_k, route_mode, type, ld, stride_s);
    if (rc) return rc;
    if (d_grad_logits && (ld_grad < E || (S > 1 && stride_grad_s < (L > 0 ? (L - 1) * ld_grad + E : 0)))) return -2;
    if (S == 0) return 0;
    if (!d_loss || !d_counts || !d_prob || !d_tokens || (L > 0 && (!d_logits || !d_topk_idx))) return -1;
    const int size = type == CHIMERE_TYPE_F32 ? 4 : 2;
    if (misaligned(d_ws, 256) || misaligned(d_logits, size) || misaligned(d_grad_logits, size) || misaligned(d_topk_idx, 4) || misaligned(d_loss, 4) || misaligned(d_counts, 4) ||
        misaligned(d_prob, 4) || misaligned(d_tokens, 4) || misaligned(d_grad_loss, 4)) return -5;
    const Plan plan = plan_of(S, (int)L, top_k);
    const Scratch a = scratch_of(plan, S, E);
    if (a.total && !d_ws) return -1;
    if (ws_bytes < a.total) return -4;
    uint8_t* ws = (uint8_t*)d_ws;
    BalanceParams p{};
    p.logits = d_logits; p.ld = ld; p.stride_s = stride_s; p.ids = d_topk_idx ? d_topk_idx : d_counts;   /* (no tokens: not read) */ p.mask = d_mask;
    p.S = (int)S; p.L = (int)L; p.E = E; p.k = top_k; p.mode = route_mode; p.coef = coef;
    p.loss = d_loss; p.counts = d_counts; p.prob = d_prob; p.tokens = d_tokens;
    p.d_loss = d_grad_loss; p.d_logits = d_grad_logits; p.ldd = ld_grad; p.stride_ds = stride_grad_s;
    p.vec = vectors(d_logits, ld, S > 1 ? stride_s : 0, E, type) && (!d_grad_logits || vectors(d_grad_logits, ld_grad, S > 1 ? stride_grad_s : 0, E, type));
    p.pieces = plan.pieces; p.rows = plan.rows; p.count_pieces = plan.count_pieces; p.count_rows = plan.count_rows;
    p.count_part = (int32_t*)(ws + a.count_part); p.part = (float*)(ws + a.part); p.group_part = (double*)(ws + a.group_part); p.counters = (int32_t*)(ws + a.counters);
    if (p.count_pieces) {
        count_kernel<<<(unsigned)(S * p.count_pieces * kB_CountCluster), kB_Threads, 0, stream>>>(p);
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return rc_of(e);
    }
    return rc_of(launch_balance(p, type, stream));
}

int chimere_b200_balance_loss_backward(const void* d_logits, int type, int64_t ld, int64_t stride_s, const uint8_t* d_mask, const int32_t* d_counts, const int32_t* d_tokens,
                                       int64_t S, int64_t L, int E, int top_k, int route_mode, float coef, const float* d_grad_loss, void* d_grad_logits, int64_t ld_grad,
                                       int64_t stride_grad_s, cudaStream_t stream) {
    const int rc = check_dims(S, L, E, top_k, route_mode, type, ld, stride_s);
    if (rc) return rc;
    if (ld_grad < E || (S > 1 && stride_grad_s < (L > 0 ? (L - 1) * ld_grad + E : 0))) return -2;
    if (S == 0 || L == 0) return 0;
    if (!d_logits || !d_counts || !d_tokens || !d_grad_logits) return -1;
    const int size = type == CHIMERE_TYPE_F32 ? 4 : 2;
    if (misaligned(d_logits, size) || misaligned(d_grad_logits, size) || misaligned(d_counts, 4) || misaligned(d_tokens, 4) || misaligned(d_grad_loss, 4)) return -5;
    const Plan plan = plan_of(S, (int)L, top_k);
    BalanceParams p{};
    p.logits = d_logits; p.ld = ld; p.stride_s = stride_s; p.mask = d_mask;
    p.S = (int)S; p.L = (int)L; p.E = E; p.k = top_k; p.mode = route_mode; p.coef = coef;
    p.counts = const_cast<int32_t*>(d_counts); p.tokens = const_cast<int32_t*>(d_tokens);
    p.d_loss = d_grad_loss; p.d_logits = d_grad_logits; p.ldd = ld_grad; p.stride_ds = stride_grad_s;
    p.vec = vectors(d_logits, ld, S > 1 ? stride_s : 0, E, type) && vectors(d_grad_logits, ld_grad, S > 1 ? stride_grad_s : 0, E, type);
    p.pieces = plan.pieces; p.rows = plan.rows;
    return rc_of(launch_balance(p, type, stream));
}

}  // extern "C"
