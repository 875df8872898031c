// w8a8.cu -- products of 8-bit integers with a scale per token and a scale per channel, dense and grouped by expert, and the rows
// that go into them (sm_100a).
//
// Math:   quantised row     scale = max|x| / 127,  q = rint(x / scale)
//         product           y[m][n] = act( (sum_k xq[m][k] * wq[n][k]) * sx[m] * sw[n] + bias[n] )
// The sums are exact (int32; |sum| <= 128 * 128 * K < 2^31 for K <= 131071), everything behind them is fp32, and the result is rounded
// once to the output's type.
// Rows, scales and activations are read by ordinary loads: within a call the kernel in front may still be writing them when a grid starts, so they are no read-only
// data of that grid.  The weights are, and go past the L1 cache by non-coherent loads or by TMA.
#include <cuda.h>
#include <cuda_bf16.h>

#include <type_traits>

#include "common.cuh"
#include "kernels.h"

namespace chimere {
namespace {

constexpr int kF32 = CHIMERE_TYPE_F32, kF16 = CHIMERE_TYPE_F16, kBF16 = CHIMERE_TYPE_BF16;
constexpr int kMaxGroups = 1024;
constexpr int kMaxK = 131071;
constexpr int64_t kMaxRows = 0x7FFFFF00;   // of a product: a tile's last row, filled up, is counted in 32 bits

// ------------------------------------------------------------------ rows -> int8 ----
// A row by GROUP threads, which keep it as it came (16 bytes of kQ_Vecs pieces each) between the maximum and the division, so that it is read
// once; what a row has beyond that is read again, from L2.  Bound: memory, so what counts is how many rows are on their way at a time: one warp
// per row where rows are short and many (no barrier, nothing waits for another row), a CTA per row else.
struct QuantParams {
    const void* x;
    int64_t ldx;
    int64_t x_rows;
    const int32_t* rows;   // or null
    int rows_div;
    int K;
    int8_t* q;
    int64_t ldq;
    float* scale;
    int64_t M;
    int vec;               // x rows start on 16-byte boundaries
};

template <int TYPE> struct Elem {   // eight values as they lie in memory
    static constexpr int kWords = TYPE == kF32 ? 8 : 4;
    using T = typename std::conditional<TYPE == kF32, float, uint16_t>::type;
    struct Raw { uint32_t w[kWords]; };
    __device__ static __forceinline__ Raw load8(const T* p) {
        Raw r;
#pragma unroll
        for (int i = 0; i < kWords / 4; ++i) {
            const uint4 a = reinterpret_cast<const uint4*>(p)[i];
            r.w[4 * i] = a.x; r.w[4 * i + 1] = a.y; r.w[4 * i + 2] = a.z; r.w[4 * i + 3] = a.w;
        }
        return r;
    }
    __device__ static __forceinline__ float of(uint32_t bits) { return TYPE == kF16 ? h2f(bits) : __uint_as_float(bits << 16); }
    __device__ static __forceinline__ float value(const Raw& r, int i) {
        if (TYPE == kF32) return __uint_as_float(r.w[i % kWords]);
        if (TYPE == kBF16 && (i & 1)) return __uint_as_float(r.w[i / 2] & 0xFFFF0000u);
        return of((r.w[i / 2] >> (16 * (i & 1))) & 0xFFFFu);
    }
    __device__ static __forceinline__ float one(const T* p) {
        if constexpr (TYPE == kF32) return *p;
        else return of(*p);
    }
    // bits of the largest magnitude: patterns of non-negative floats order like the values, with the NaNs above infinity
    __device__ static __forceinline__ uint32_t top(const Raw& r, uint32_t m) {
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(value(r, i)) & 0x7FFFFFFFu);
        return m;
    }
};

// The two quotients.  In the wide range of magnitudes both come correctly rounded from a reciprocal (div_by_recip), in rows outside it from the
// division operator; a scale below the normal numbers would make the quotients coarse, so it stays at 2^-126.
// Nearest integer, ties to even: the sum with 1.5 * 2^23 holds it in its low byte (|x / scale| <= 127.5).
struct RowScale {
    float scale, recip;
    __device__ __forceinline__ static bool wide(float amax) { return amax > 1e-25f && amax < 1e25f; }
    __device__ __forceinline__ explicit RowScale(float amax) {
        scale = div_by_recip(amax, 127.0f, 1.0f / 127.0f);
        recip = __frcp_rn(scale);
    }
    __device__ __forceinline__ uint32_t q(float x) const { return __float_as_uint(__fadd_rn(div_by_recip(x, scale, recip), 12582912.0f)); }
    // two at a time: the same operations as div_by_recip's, each rounded like the scalar form
    __device__ __forceinline__ uint32_t q2(float a, float b) const {
        const uint64_t x = pack2f(a, b), r = pack2f(recip, recip), s = pack2f(-scale, -scale);
        uint64_t v = mul2(x, r);
        v = fma2(fma2(v, s, x), r, v);
        v = add2(fma2(fma2(v, s, x), r, v), pack2f(12582912.0f, 12582912.0f));
        return prmt((uint32_t)v, (uint32_t)(v >> 32), 0x0040u);
    }
    __device__ __forceinline__ uint32_t q4(float a, float b, float c, float d) const { return prmt(q2(a, b), q2(c, d), 0x5410u); }
};

// GROUP 32: a warp per row; GROUP 0: a CTA per row.  VEC: rows on 16-byte boundaries
template <int TYPE, int GROUP, int VECS, bool VEC = true>
__global__ void __launch_bounds__(GROUP ? 256 : 1024) quantize_rows_kernel(QuantParams p) {
    using E = Elem<TYPE>;
    __shared__ uint32_t s_max[32];
    const int tid = GROUP ? threadIdx.x % 32 : threadIdx.x, nt = GROUP ? 32 : blockDim.x;
    griddep_wait();          // (in front of the next kernel's start: what lies before this kernel is then complete for that one too)
    griddep_launch();
    const int64_t row = GROUP ? (int64_t)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32 : blockIdx.x;
    if (GROUP && row >= p.M) return;
    int64_t src = row;
    if (p.rows) {
        const int32_t r = p.rows[row];
        src = r < 0 ? -1 : r / p.rows_div;
    }
    int8_t* q = p.q + row * p.ldq;
    if (src < 0 || src >= p.x_rows) {   // no such row: zeros
        for (int i = tid; i < p.K; i += nt) q[i] = 0;
        if (tid == 0) p.scale[row] = 0.0f;
        return;
    }
    const typename E::T* x = reinterpret_cast<const typename E::T*>(p.x) + src * p.ldx;
    uint32_t m = 0;
    constexpr int kOnes = VEC ? 1 : 16;   // rows off the 16-byte boundaries: value by value
    float one[kOnes];
    if (!VEC) {
#pragma unroll
        for (int i = 0; i < kOnes; ++i) one[i] = tid + i * nt < p.K ? E::one(x + tid + i * nt) : 0.0f;
#pragma unroll
        for (int i = 0; i < kOnes; ++i) m = max(m, __float_as_uint(one[i]) & 0x7FFFFFFFu);
    }
    const int nv = VEC ? p.K >> 3 : 0, ones = VEC ? 8 * nv : min(p.K, kOnes * nt);
    typename E::Raw v[VECS];
#pragma unroll
    for (int i = 0; i < VECS; ++i)
        if (tid + i * nt < nv) v[i] = E::load8(x + 8 * (tid + i * nt));
#pragma unroll
    for (int i = 0; i < VECS; ++i)
        if (tid + i * nt < nv) m = E::top(v[i], m);
    for (int i = tid + VECS * nt; i < nv; i += nt) m = E::top(E::load8(x + 8 * i), m);
    for (int i = ones + tid; i < p.K; i += nt) m = max(m, __float_as_uint(E::one(x + i)) & 0x7FFFFFFFu);
    m = __reduce_max_sync(0xffffffffu, m);
    if (!GROUP && nt > 32) {
        if ((tid & 31) == 0) s_max[tid >> 5] = m;
        __syncthreads();
        m = __reduce_max_sync(0xffffffffu, (tid & 31) < (nt >> 5) ? s_max[tid & 31] : 0u);
    }
    if (m >= 0x7F800000u) {   // an infinity or a NaN in the row: the whole row of the product becomes NaN
        for (int i = tid; i < p.K; i += nt) q[i] = 0;
        if (tid == 0) p.scale[row] = __uint_as_float(0x7FC00000u);
        return;
    }
    const float amax = __uint_as_float(m);
    if (!RowScale::wide(amax)) {
        const float scale = amax == 0.0f ? 0.0f : fmaxf(amax / 127.0f, 1.17549435e-38f);
#pragma unroll 1
        for (int i = tid; i < p.K; i += nt) q[i] = (int8_t)(scale == 0.0f ? 0 : __float2int_rn(E::one(x + i) / scale));
        if (tid == 0) p.scale[row] = scale;
        return;
    }
    const RowScale s(amax);
    if (tid == 0) p.scale[row] = s.scale;
    auto put = [&](int i, const typename E::Raw& w) {
        uint2 o;
        o.x = s.q4(E::value(w, 0), E::value(w, 1), E::value(w, 2), E::value(w, 3));
        o.y = s.q4(E::value(w, 4), E::value(w, 5), E::value(w, 6), E::value(w, 7));
        *reinterpret_cast<uint2*>(q + 8 * i) = o;
    };
#pragma unroll
    for (int i = 0; i < VECS; ++i)
        if (tid + i * nt < nv) put(tid + i * nt, v[i]);
    for (int i = tid + VECS * nt; i < nv; i += nt) put(i, E::load8(x + 8 * i));
    if (!VEC) {
#pragma unroll
        for (int i = 0; i < kOnes; ++i)
            if (tid + i * nt < p.K) q[tid + i * nt] = (int8_t)s.q(one[i]);
    }
    for (int i = ones + tid; i < p.K; i += nt) q[i] = (int8_t)s.q(E::one(x + i));
}

// Row i of (q, scale) = row rows[i] / rows_div of (from, from_scale), a warp each; 16 bytes at a time (what lies behind a row's K values goes along).
__global__ void __launch_bounds__(256) gather_rows_kernel(const int8_t* from, const float* from_scale, int64_t from_rows, const int32_t* rows, int rows_div, int8_t* q, float* scale,
                                                          int64_t M, int64_t ld) {
    griddep_wait();
    griddep_launch();
    const int64_t i = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
    const int lane = threadIdx.x % 32;
    if (i >= M) return;
    const int32_t r = rows[i];
    const int64_t src = r < 0 ? -1 : r / rows_div;
    const bool there = src >= 0 && src < from_rows;
    const uint4* a = reinterpret_cast<const uint4*>(from + (there ? src : 0) * ld);
    uint4* b = reinterpret_cast<uint4*>(q + i * ld);
    const int n = (int)(ld / 16);
    for (int j = lane; j < n; j += 128) {
        uint4 v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = j + 32 * u < n && there ? a[j + 32 * u] : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int u = 0; u < 4; ++u) if (j + 32 * u < n) b[j + 32 * u] = v[u];
    }
    if (lane == 0) scale[i] = there ? from_scale[src] : 0.0f;
}

template <int TYPE>
cudaError_t launch_quantize_type(const QuantParams& p, cudaStream_t stream, bool pdl) {
    auto go = [&](auto kernel, int64_t grid, int nt) -> cudaError_t {
        if (pdl) return launch_pdl(kernel, dim3((unsigned)grid), nt, 0, stream, p);
        kernel<<<(unsigned)grid, nt, 0, stream>>>(p);
        return cudaGetLastError();
    };
    // A warp holds 512 bytes of a row per register piece (four registers); sixteen of them at most, and enough rows for every SM's warps.
    const int pieces = (p.K / 8 * (TYPE == kF32 ? 2 : 1) + 31) / 32;
    if (p.vec && pieces <= 16 && p.M >= 148 * 8) {
        constexpr int k = TYPE == kF32 ? 2 : 1;
        constexpr int kRows = 4;   // (8192 x 4096 bf16 20.5 us, with eight 21.6; 32768 x 512 f32 14.4, with eight 15.4, with two 18.5)
        const int64_t grid = (p.M + kRows - 1) / kRows;
        if (pieces <= 4) return go(quantize_rows_kernel<TYPE, 32, 4 / k>, grid, 32 * kRows);
        if (pieces <= 8) return go(quantize_rows_kernel<TYPE, 32, 8 / k>, grid, 32 * kRows);
        return go(quantize_rows_kernel<TYPE, 32, 16 / k>, grid, 32 * kRows);
    }
    // sixteen values per thread, at least a warp
    int nt = (p.K + 15) / 16;
    nt = nt > 1024 ? 1024 : (nt + 31) / 32 * 32;
    return p.vec ? go(quantize_rows_kernel<TYPE, 0, 2>, p.M, nt) : go(quantize_rows_kernel<TYPE, 0, 2, false>, p.M, nt);
}
cudaError_t launch_quantize(QuantParams p, int type, cudaStream_t stream, bool pdl) {
    p.vec = ((uintptr_t)p.x & 15) == 0 && (p.ldx * (type == kF32 ? 4 : 2)) % 16 == 0;
    return type == kF32 ? launch_quantize_type<kF32>(p, stream, pdl) : type == kF16 ? launch_quantize_type<kF16>(p, stream, pdl) : launch_quantize_type<kBF16>(p, stream, pdl);
}

// ------------------------------------------------------------------ product ----
// tcgen05 kind::i8; operands by TMA as rows of 128 bytes (128-byte swizzle), zeros beyond K and beyond the last row.  Two kernels, which differ
// in whose rows are the MMA's:
//   few tokens (matmul_kernel)   128 weight rows (two such blocks, gate and up, where the activation joins them) x BN tokens, BN the narrowest of
//       16, 32 and 64 that suits the batch.  Where there are fewer tiles than SMs a cluster of up to eight CTAs shares a tile, each with a
//       part of K; their int32 sums meet in shared memory over the cluster, exact in any order.
//   many tokens (wide_kernel)    256 tokens x 256 weight rows by a pair of CTAs (cta_group::2): each fetches its 128 tokens and 128 of the weight rows
//       (with SwiGLU one the gate's, the other the up matrix'), half of what a CTA alone would need for the same MMAs.  A thread of the epilogue has
//       one token's row: its scale and place are looked up once, its results go out 32 bytes at a time.
// Bound: the weights' bytes where experts or a matrix have few tokens (gate and up of 104 experts of 512 x 2048, 128 pairs: 38 us, 5.6 TB/s; 128 of 1856 x 2688, 1998
// pairs: 104 us, 6.1 TB/s), the tensor pipe in large batches (8192 tokens x 8192 of 4096: 159 us, 3.46 POP/s, the pipe 94 % active; a CTA alone per tile 313), what goes through
// L2 where K is small (32768 pairs x 2048 of 512: 70 us).
// All waits are bounded: one that runs out makes the tile's outputs NaN and raises the status word.
constexpr int kMM_KBytes = 128;          // of K per stage
constexpr int kMM_ABytes = 128 * kMM_KBytes;
constexpr int kMM_MaxStages = 12;
constexpr int kMM_Threads = 384, kMM_FirstEpi = 4;   // warps 0 TMA, 1 MMA, 4 .. 11 epilogue (2 and 3 help to set up)

struct MatmulParams {
    const float* sx;
    const float* sw;
    const float* bias;
    void* y;
    int64_t ldy, y_rows;
    const int32_t* offsets;    // grouped: [E + 1], else null
    const int32_t* out_rows;   // or null
    int32_t* status;           // or null
    int M, N, K, E;
    int y_type, act;
    int mt, nt;                // dense: token tiles; tiles of outputs
    int n_stages, split;
    int early;                 // the weights, scales and offsets do not come from the previous kernel
    int vec;                   // wide: rows of y start on 32-byte boundaries
};

struct Tile { int expert, row0, ntok, n0; };

// Token tiles per expert, summed over the experts in front, and where the experts' rows start.
struct GroupTable {
    int prefix[kMaxGroups + 1], start[kMaxGroups + 1];
    int scan[32];
};

__device__ __forceinline__ bool elect1() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
template <int CTAS>
__device__ __forceinline__ void commit(uint64_t* bar) {   // ... to the barrier at this place in both CTAs of a pair
    if (CTAS == 1) asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
    else asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)), "h"((uint16_t)3) : "memory");
}
template <int CTAS>
__device__ __forceinline__ void mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if (CTAS == 1)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __host__ constexpr uint32_t idesc_i8(int m, int n) { return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24); }
template <int CTAS>
__device__ __forceinline__ void tmem_alloc(uint32_t* where, uint32_t cols) {
    if (CTAS == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(where)), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(where)), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
}
template <int CTAS>
__device__ __forceinline__ void tmem_free(uint32_t tmem, uint32_t cols) {
    if (CTAS == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols) : "memory");
}
// rows of 128 bytes, 128-byte swizzle: groups of eight rows 1024 bytes apart; a step of 32 along K is 32 bytes of the start address
__device__ __forceinline__ uint64_t desc_sw128(uint32_t saddr) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | (1ull << 16) | ((uint64_t)(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// CTAS 2: the copy lands in this CTA and is counted on the barrier at this place in the pair's first CTA
template <int CTAS> __device__ __forceinline__ uint32_t bar_addr(uint64_t* bar) { return CTAS == 1 ? smem_u32(bar) : smem_u32(bar) & 0xFEFFFFFFu; }
template <int CTAS>
__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    if (CTAS == 1)
        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                     ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
    else
        asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                     ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
template <int CTAS>
__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    if (CTAS == 1)
        asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                     ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
    else
        asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                     ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }
// TMEM -> registers, thread = lane, neighbouring columns (the wait in the same statement: no use of a value can move in front of it)
__device__ __forceinline__ void ld16(uint32_t taddr, int* v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
          "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_addr(uint32_t saddr, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
    return r;
}
__device__ __forceinline__ int ld_cluster(uint32_t addr) {
    int v;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void ld_cluster4(uint32_t addr, int (&sum)[4]) {   // added to four sums
    int v[4];
    asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(addr) : "memory");
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i] += v[i];
}
// An arrival that orders nothing but what the tensor-memory fence in front of it does: with the cluster's release it would wait for the tile's stores to
// reach L2 (a microsecond per tile).
__device__ __forceinline__ void arrive_cluster(uint32_t addr) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}

// By all threads; returns the call's token tiles.
template <int TOKENS, int THREADS>
__device__ __forceinline__ int group_table(const MatmulParams& p, GroupTable& g) {
    constexpr int kPer = (kMaxGroups + THREADS) / THREADS;   // (the table's end included)
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int mine[kPer], start[kPer], sum = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int e = tid * kPer + i;
        mine[i] = start[i] = 0;
        if (e < p.E) {
            start[i] = min(max(p.offsets[e], 0), p.M);
            mine[i] = (min(max(p.offsets[e + 1], start[i]), p.M) - start[i] + TOKENS - 1) / TOKENS;
        }
        sum += mine[i];
    }
    int scan = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, scan, d);
        if (lane >= d) scan += o;
    }
    if (lane == 31) g.scan[warp] = scan;
    __syncthreads();
    int before = scan - sum;
    for (int w = 0; w < warp; ++w) before += g.scan[w];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int e = tid * kPer + i;
        if (e <= p.E) { g.prefix[e] = before; g.start[e] = start[i]; }
        before += mine[i];
    }
    __syncthreads();
    return g.prefix[p.E];
}

// Tile `id` of the call: token tiles fastest, so that the CTAs at work at a time share weight rows.
template <int TOKENS, int OUTS>
__device__ __forceinline__ Tile take_tile(const MatmulParams& p, const GroupTable& g, int id) {
    Tile t;
    if (!p.offsets) {
        const int m = id % p.mt;
        t.expert = 0;
        t.row0 = m * TOKENS;
        t.ntok = min(TOKENS, p.M - t.row0);
        t.n0 = id / p.mt * OUTS;
        return t;
    }
    // prefix[e]: token tiles of the experts in front of e; largest e with prefix[e] * nt <= id
    const int tile = id / p.nt;
    int lo = 0, hi = p.E - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (g.prefix[mid] <= tile) lo = mid; else hi = mid - 1;
    }
    const int c = g.prefix[lo + 1] - g.prefix[lo], local = id - g.prefix[lo] * p.nt, m = local % c, start = g.start[lo];
    t.expert = lo;
    t.row0 = start + m * TOKENS;
    t.ntok = min(TOKENS, min(max(p.offsets[lo + 1], start), p.M) - t.row0);
    t.n0 = local / c * OUTS;
    return t;
}
template <int TYPE> struct Out;
template <> struct Out<kF32> {
    using T = float;
    __device__ static __forceinline__ T of(float v) { return v; }
};
template <> struct Out<kF16> {
    using T = __half;
    __device__ static __forceinline__ T of(float v) { return __float2half_rn(v); }
};
template <> struct Out<kBF16> {
    using T = __nv_bfloat16;
    __device__ static __forceinline__ T of(float v) { return __float2bfloat16_rn(v); }
};
__device__ __forceinline__ void put(const MatmulParams& p, int64_t at, float v) {
    if (p.y_type == kF32) reinterpret_cast<float*>(p.y)[at] = v;
    else if (p.y_type == kBF16) reinterpret_cast<__nv_bfloat16*>(p.y)[at] = Out<kBF16>::of(v);
    else reinterpret_cast<__half*>(p.y)[at] = Out<kF16>::of(v);
}
// (the channel's scale first: a token's may lie anywhere in fp32's range, and then only a result that does not fit overflows)
__device__ __forceinline__ float scaled(int acc, float sw, float sx, float b) { return __fmaf_rn(__fmul_rn((float)acc, sw), sx, b); }
__device__ __forceinline__ float relu2(float v) { v = v > 0.0f || v != v ? v : 0.0f; return v * v; }

// what one thread needs of its weight row(s)
struct Channel { float sw, sw_up, b, b_up; };
__device__ __forceinline__ Channel channel(const MatmulParams& p, bool dual, int expert, int n) {
    Channel c{0.0f, 0.0f, 0.0f, 0.0f};
    if (n < p.N) {
        const int64_t at = (int64_t)expert * (dual ? 2 * (int64_t)p.N : p.N) + n;
        c.sw = p.sw[at];
        if (p.bias) c.b = p.bias[at];
        if (dual) {
            c.sw_up = p.sw[at + p.N];
            if (p.bias) c.b_up = p.bias[at + p.N];
        }
    }
    return c;
}
// silu(g) * u for two pairs: g / (1 + exp(-g)), exp as 2^h times 1 + r with h = -g log2(e) rounded and r what the rounding left out (ln(2) in two parts), the
// quotient with the hardware's reciprocal.  From g = -87 on silu is off by ten half-steps of fp32 at most: ex2 four, 1 + r and its product two, 1 + exp one, the
// reciprocal two, the last product one.  Below about -87.3 the denominator passes 2^126, its reciprocal is subnormal and comes out as 0, and so does silu: off by less than
// 88 * 2^-126.  (Through expf and the division operator the epilogue took longer than the MMAs: 32768 tokens x 512 of
// 2048 122 us, plain results of the same sums 59.)
__device__ __forceinline__ void silu_mul2(float g0, float g1, float u0, float u1, float (&y)[2]) {
    float a = -g0, b = -g1;
    asm("min.NaN.f32 %0, %0, %1;\n\tmax.NaN.f32 %0, %0, %2;" : "+f"(a) : "f"(200.0f), "f"(-200.0f));   // (beyond, exp is infinite or 0 as it is there)
    asm("min.NaN.f32 %0, %0, %1;\n\tmax.NaN.f32 %0, %0, %2;" : "+f"(b) : "f"(200.0f), "f"(-200.0f));
    const uint64_t x = pack2f(a, b), h = mul2(x, pack2f(1.44269504f, 1.44269504f)), one = pack2f(1.0f, 1.0f);
    uint64_t r = fma2(h, pack2f(-0.693147182f, -0.693147182f), x);
    r = fma2(h, pack2f(1.90465421e-9f, 1.90465421e-9f), r);
    unpack2(h, a, b);
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(a));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(b));
    unpack2(add2(mul2(pack2f(a, b), add2(r, one)), one), a, b);
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(a));
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(b));
    unpack2(mul2(mul2(pack2f(g0, g1), pack2f(a, b)), pack2f(u0, u1)), y[0], y[1]);
}
// two tokens of one channel
template <bool DUAL>
__device__ __forceinline__ void finish2(const MatmulParams& p, const Channel& c, float sx0, float sx1, int a0, int a1, int up0, int up1, float (&o)[2]) {
    o[0] = scaled(a0, c.sw, sx0, c.b);
    o[1] = scaled(a1, c.sw, sx1, c.b);
    if (DUAL) silu_mul2(o[0], o[1], scaled(up0, c.sw_up, sx0, c.b_up), scaled(up1, c.sw_up, sx1, c.b_up), o);
    else if (p.act == CHIMERE_ACT_RELU2) { o[0] = relu2(o[0]); o[1] = relu2(o[1]); }
}

struct MatmulShared {
    uint64_t full[kMM_MaxStages], empty[kMM_MaxStages];
    uint64_t tfull[2], tempty[2];
    uint64_t drain;
    uint32_t tmem_base;
    int failed;
    float sx[2][64];   // of a tile's tokens: scale and row of y
    int row[2][64];
};

template <int BN, bool DUAL>
__global__ void __launch_bounds__(kMM_Threads) matmul_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, MatmulParams p) {
    constexpr uint32_t kStage = kMM_ABytes * (DUAL ? 2 : 1) + BN * kMM_KBytes;
    constexpr uint32_t kAccCols = BN * (DUAL ? 2 : 1);
    constexpr uint32_t kTmemCols = kAccCols * 2 < 32 ? 32 : kAccCols * 2;
    static_assert(kTmemCols <= 512, "two accumulators fit");
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) MatmulShared sh;
    __shared__ GroupTable table;
    uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const int S = p.split, rank = S > 1 ? blockIdx.x % S : 0, first = blockIdx.x / S, step = gridDim.x / S;
    const uint32_t stages = smem_u32(smem);

    if (tid == 0) { prefetch_map(&map_w); prefetch_map(&map_x); }
    if (!p.early) griddep_wait();
    const int total = (p.offsets ? group_table<BN, kMM_Threads>(p, table) : p.mt) * p.nt;
    if (first >= total) {   // (the whole cluster; nothing has been allocated)
        griddep_launch();
        griddep_wait();   // (whoever waits for this grid has what lies before it as well)
        return;
    }

    if (tid == 0) {
        for (int i = 0; i < p.n_stages; ++i) { mbar_init(&sh.full[i], 1); mbar_init(&sh.empty[i], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&sh.tfull[i], 1); mbar_init(&sh.tempty[i], 4); }
        mbar_init(&sh.drain, 1);
        sh.failed = 0;
        mbar_fence_init();
    }
    if (warp == 1) tmem_alloc<1>(&sh.tmem_base, kTmemCols);
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = sh.tmem_base;
    if (tid == 0) griddep_launch();

    const int nkb = (p.K + kMM_KBytes - 1) / kMM_KBytes;
    const int kb0 = (int)((int64_t)rank * nkb / S), kb1 = (int)((int64_t)(rank + 1) * nkb / S);

    if (warp == 0) {
        int st = 0;
        uint32_t ph = 0, used = 0;
        bool ok = true, waited = !p.early;
        for (int id = first; ok && id < total; id += step) {
            const Tile t = take_tile<BN, 128>(p, table, id);
            for (int kb = kb0; kb < kb1; ++kb) {
                if (!mbar_wait(&sh.empty[st], ph ^ 1u)) { ok = false; break; }
                const uint32_t dst = stages + st * kStage, bar = smem_u32(&sh.full[st]);
                if (elect1()) {
                    mbar_expect_tx(&sh.full[st], kStage);
                    tma_3d<1>(dst, &map_w, kb * kMM_KBytes, t.n0, t.expert, bar);
                    if (DUAL) tma_3d<1>(dst + kMM_ABytes, &map_w, kb * kMM_KBytes, p.N + t.n0, t.expert, bar);
                }
                __syncwarp();
                if (!waited) { griddep_wait(); waited = true; }
                if (elect1()) tma_2d<1>(dst + kMM_ABytes * (DUAL ? 2 : 1), &map_x, kb * kMM_KBytes, t.row0, bar);
                __syncwarp();
                used |= 1u << st;
                if (++st == p.n_stages) { st = 0; ph ^= 1u; }
            }
        }
        if (!ok) {   // the copies under way land before the CTA goes
            sh.failed = 1;
            for (int i = 0; i < p.n_stages; ++i)
                if (used >> i & 1u) mbar_wait(&sh.full[i], (i < st ? ph : ph ^ 1u));
        }
    } else if (warp == 1) {
        constexpr uint32_t idesc = idesc_i8(128, BN);
        int st = 0, n = 0;
        uint32_t ph = 0;
        bool ok = true;
        for (int id = first; ok && id < total; id += step, ++n) {
            const int buf = n & 1;
            if (!mbar_wait(&sh.tempty[buf], ((n >> 1) & 1) ^ 1u)) { ok = false; break; }
            fence_after();
            const uint32_t d = tmem + buf * kAccCols;
            for (int kb = kb0; kb < kb1; ++kb) {
                if (!mbar_wait(&sh.full[st], ph)) { ok = false; break; }
                fence_after();
                if (elect1()) {
                    const uint32_t a = stages + st * kStage, b = a + kMM_ABytes * (DUAL ? 2 : 1);
#pragma unroll
                    for (int k = 0; k < kMM_KBytes / 32; ++k) {
                        const uint32_t acc = kb > kb0 || k > 0;
                        mma_i8<1>(d, desc_sw128(a + 32 * k), desc_sw128(b + 32 * k), idesc, acc);
                        if (DUAL) mma_i8<1>(d + BN, desc_sw128(a + kMM_ABytes + 32 * k), desc_sw128(b + 32 * k), idesc, acc);
                    }
                    commit<1>(&sh.empty[st]);
                }
                __syncwarp();
                if (++st == p.n_stages) { st = 0; ph ^= 1u; }
            }
            if (ok && elect1()) commit<1>(&sh.tfull[buf]);
            __syncwarp();
        }
        if (!ok) {
            sh.failed = 1;
            if (elect1()) commit<1>(&sh.drain);   // (the MMAs under way)
            __syncwarp();
            mbar_wait(&sh.drain, 0);
        }
    } else if (warp >= kMM_FirstEpi) {
        // four warps take every other tile, and look up a tile's scales and places while the one before is on its way
        const int q = warp & 3, buf = (warp - kMM_FirstEpi) >> 2, row = q * 32 + lane;
        const uint32_t taddr = tmem + ((uint32_t)(q * 32) << 16) + buf * kAccCols;
        bool ok = true;
        griddep_wait();   // (the tokens' scales; and nothing of y is written before what used its memory has ended)
        Tile t;
        Channel ch;
        float sx = 0.0f;
        int to = -1;
        static_assert(BN <= 128, "a token per thread");
        auto look_up = [&](int id) {
            t = take_tile<BN, 128>(p, table, id);
            ch = channel(p, DUAL, t.expert, t.n0 + row);
            if (row < t.ntok) {
                sx = p.sx[t.row0 + row];
                to = p.out_rows ? p.out_rows[t.row0 + row] : t.row0 + row;
            }
        };
        int id = first + buf * step;
        if (id < total && S == 1) look_up(id);
        uint32_t ph = 0;
        for (; id < total; id += 2 * step, ph ^= 1u) {
            if (S > 1) {   // this CTA's part of the sums, over the operands' buffers: [gate / up][token][128]
                t = take_tile<BN, 128>(p, table, id);
                if (!mbar_wait(&sh.tfull[buf], ph)) sh.failed = 1;
                fence_after();
                int* part = reinterpret_cast<int*>(smem);
                for (int c0 = 0; c0 < t.ntok; c0 += 16)
#pragma unroll
                    for (int h = 0; h < (DUAL ? 2 : 1); ++h) {
                        int v[16];
                        ld16(taddr + h * BN + c0, v);
#pragma unroll
                        for (int j = 0; j < 16; ++j) part[(h * BN + c0 + j) * 128 + row] = v[j];
                    }
                fence_before();
                break;
            }
            asm volatile("bar.sync %0, 128;" ::"r"(1 + buf) : "memory");   // (the tile before has been read)
            if (row < t.ntok) { sh.sx[buf][row] = sx; sh.row[buf][row] = to; }
            asm volatile("bar.sync %0, 128;" ::"r"(1 + buf) : "memory");
            const Channel c = ch;
            const int ntok = t.ntok, n = t.n0 + row;
            if (id + 2 * step < total) look_up(id + 2 * step);
            if (ok && !mbar_wait(&sh.tfull[buf], ph)) { ok = false; sh.failed = 1; }
            fence_after();
            for (int c0 = 0; c0 < ntok; c0 += 16) {
                int v[16], u[16];
                ld16(taddr + c0, v);
                if (DUAL) ld16(taddr + BN + c0, u);
#pragma unroll
                for (int j = 0; j < 16; j += 2) {
                    float o[2];
                    const int m = c0 + j;
                    finish2<DUAL>(p, c, sh.sx[buf][m], sh.sx[buf][m + 1], v[j], v[j + 1], DUAL ? u[j] : 0, DUAL ? u[j + 1] : 0, o);
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        if (m + i < ntok && n < p.N) {
                            const int64_t r = sh.row[buf][m + i];
                            if (r >= 0 && r < p.y_rows) put(p, r * p.ldy + n, ok ? o[i] : __uint_as_float(0x7FC00000u));
                        }
                }
            }
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cta(&sh.tempty[buf]);
        }
    }
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == 1) tmem_free<1>(tmem, kTmemCols);   // (in front of the cluster's barrier: who waits for a neighbour holds none)
    if (S > 1) {
        const Tile t = take_tile<BN, 128>(p, table, first);
        griddep_wait();
        Channel ch[4];   // of this thread's four neighbouring outputs, the same for all of its tokens (384 is a multiple of 32)
#pragma unroll
        for (int j = 0; j < 4; ++j) ch[j] = channel(p, DUAL, t.expert, t.n0 + 4 * (tid & 31) + j);
        cluster_sync();   // every part is there
        bool bad = false;
        for (int s = 0; s < S; ++s) bad |= ld_cluster(cluster_addr(smem_u32(&sh.failed), s)) != 0;
        for (int i = rank * kMM_Threads + tid; i < t.ntok * 32; i += S * kMM_Threads) {   // four neighbouring results
            const int m = i >> 5, n = t.n0 + 4 * (i & 31);
            if (n >= p.N) continue;
            int acc[4] = {}, up[4] = {};
#pragma unroll
            for (int s = 0; s < 8; ++s)   // (all on their way at once)
                if (s < S) {
                    ld_cluster4(cluster_addr(stages + 16 * i, s), acc);
                    if (DUAL) ld_cluster4(cluster_addr(stages + 16 * (i + BN * 32), s), up);
                }
            const int64_t r = p.out_rows ? p.out_rows[t.row0 + m] : t.row0 + m;
            const float sx = p.sx[t.row0 + m];
            if (r < 0 || r >= p.y_rows) continue;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float o[2];
                finish2<DUAL>(p, ch[j], sx, 0.0f, acc[j], 0, up[j], 0, o);
                if (n + j < p.N) put(p, r * p.ldy + n + j, bad ? __uint_as_float(0x7FC00000u) : o[0]);
            }
        }
        cluster_sync();   // ... and has been read
    }
    if (tid == 0 && sh.failed && p.status) atomicOr(p.status, kStatusWaitTimeout);
}

// ---- a few tokens ----
// Up to eight tokens at a time times 16 weight rows (or 16 of the gate and the same 16 of the up matrix) per warp, or per 2, 4 or 8 warps that share K in
// pieces of 64 bytes, so that each has about four of them; the sums on the warp-level int8 MMA (m16n8k32), its K order that of the bytes a lane holds: 16 neighbouring ones of a weight row and the same 16 of a token's.
// All of a warp's first weights are on their way before it looks at the tokens, which the CTA quantises itself, or the CTAs of a cluster one or two each for all of
// them (kI8: takes as they are): a call is one launch.
// Bound: the weights' bytes, and what a launch takes (1 token x 4096 of 2048: 4.6 us).  y by the formula of the other kernels, the same bits.
constexpr int kI8 = -2;                 // rows that are quantised already
constexpr int kR_Threads = 256, kR_Warps = 8, kR_Tokens = 8, kR_Units = 4;   // units of 64 bytes of K that a warp has on their way
constexpr int kR_MaxK = 8192;

struct RowsParams {
    MatmulParams m;
    const void* x;
    int64_t ldx, x_rows;
    const int32_t* rows;       // or null
    int rows_div, vec;
    const int8_t* w;
    int64_t ldw, w_plane;
    int kw;                    // warps that share K
    int cluster;               // CTAs that share the quantising of the tokens (1, 2, 4 or 8; more than one: a single group of up to eight tokens)
    int ks;                    // bytes between tokens in shared memory: 64 modulo 128, so that neighbouring tokens lie in different banks
};

__device__ __forceinline__ void mma_16832(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Grouped: blockIdx.y is a pair, whose CTAs take its expert if it is the expert's first.
template <int TYPE, bool DUAL>
__global__ void __launch_bounds__(kR_Threads) rows_kernel(const __grid_constant__ RowsParams p) {
    constexpr int TILES = DUAL ? 2 : 1;
    extern __shared__ __align__(16) int8_t xs[];          // [token][ks]
    __shared__ uint32_t s_max[kR_Tokens][kR_Warps];
    __shared__ float s_scale[kR_Tokens];
    __shared__ int s_row[kR_Tokens];
    __shared__ int red[kR_Warps][TILES][16][kR_Tokens + 1];
    __shared__ int group[3];
    const MatmulParams& mp = p.m;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int kw = p.kw, wk = warp & (kw - 1), outs = 16 * (kR_Warps / kw);
    const int C = TYPE == kI8 ? 1 : p.cluster, rank = C > 1 ? blockIdx.x & (C - 1) : 0;
    const int n0 = blockIdx.x * outs, K = mp.K, units = (K + 63) >> 6;
    if (!mp.early) griddep_wait();
    griddep_launch();
    int e = 0, start = 0, end = mp.M;
    if (mp.offsets) {
        if (tid == 0) group[0] = -1;
        __syncthreads();
        for (int i = tid; i < mp.E; i += kR_Threads) {
            const int a = min(max(mp.offsets[i], 0), mp.M), b = min(max(mp.offsets[i + 1], a), mp.M);
            if (a == (int)blockIdx.y && b > a) { group[0] = i; group[1] = a; group[2] = b; }
        }
        __syncthreads();
        e = group[0]; start = group[1]; end = group[2];
        if (e < 0) { griddep_wait(); return; }   // (whoever waits for this grid has what lies before it as well)
    }
    // this lane's rows (behind the last one: the last one again, not stored)
    const int8_t* wr[TILES][2];
#pragma unroll
    for (int i = 0; i < TILES; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int n = min(n0 + 16 * (warp / kw) + g + 8 * h, mp.N - 1) + i * mp.N;
            wr[i][h] = p.w + e * p.w_plane + n * p.ldw + 16 * t;
        }
    uint4 v[kR_Units][TILES][2];
    auto load = [&](int base) {
#pragma unroll
        for (int u = 0; u < kR_Units; ++u) {
            const int unit = base + wk + kw * u;
            const bool in = unit < units && 64 * unit + 16 * t < K && n0 < mp.N;   // (a cluster's last CTAs may have no rows)
#pragma unroll
            for (int i = 0; i < TILES; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    v[u][i][h] = make_uint4(0, 0, 0, 0);
                    if (in) asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                                         : "=r"(v[u][i][h].x), "=r"(v[u][i][h].y), "=r"(v[u][i][h].z), "=r"(v[u][i][h].w) : "l"(wr[i][h] + 64 * unit));
                }
        }
    };
    load(0);
    const Channel ch = channel(mp, DUAL, e, n0 + tid % outs);   // (a thread's results are all of one channel: 256 is a multiple of outs)
    if (mp.early) griddep_wait();

    for (int c0 = start; c0 < end; c0 += kR_Tokens) {
        const int ntok = min(kR_Tokens, end - c0);
        if (tid < ntok) s_row[tid] = mp.out_rows ? mp.out_rows[c0 + tid] : c0 + tid;
        auto source = [&](int m) -> int64_t {
            if (!p.rows) return c0 + m;
            const int r = p.rows[c0 + m], s = r < 0 ? -1 : r / p.rows_div;
            return s < p.x_rows ? s : -1;
        };
        if constexpr (TYPE == kI8) {
            for (int m = 0; m < ntok; ++m) {
                const int8_t* x = reinterpret_cast<const int8_t*>(p.x) + (int64_t)(c0 + m) * p.ldx;
                for (int i = tid; i < 4 * units; i += kR_Threads) {
                    uint4 q = make_uint4(0, 0, 0, 0);
                    if (16 * i < K) q = reinterpret_cast<const uint4*>(x)[i];
                    uint32_t* w = reinterpret_cast<uint32_t*>(&q);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {   // (nothing behind the row's last value)
                        const int left = K - 16 * i - 4 * j;
                        if (left < 4) w[j] = left <= 0 ? 0u : w[j] & (0xFFFFFFFFu >> (32 - 8 * left));
                    }
                    *reinterpret_cast<uint4*>(xs + m * p.ks + 16 * i) = q;
                }
                if (tid == 0) s_scale[m] = mp.sx[c0 + m];
            }
        } else {
            using E = Elem<TYPE>;
            const int nv = p.vec ? K >> 3 : 0;
            for (int m = rank; m < ntok; m += C) {
                const int64_t src = source(m);
                uint32_t top = 0;
                if (src >= 0) {
                    const typename E::T* x = reinterpret_cast<const typename E::T*>(p.x) + src * p.ldx;
                    for (int i = tid; i < nv; i += kR_Threads) top = E::top(E::load8(x + 8 * i), top);
                    for (int i = 8 * nv + tid; i < K; i += kR_Threads) top = max(top, __float_as_uint(E::one(x + i)) & 0x7FFFFFFFu);
                }
                top = __reduce_max_sync(0xffffffffu, top);
                if (lane == 0) s_max[m][warp] = top;
            }
            __syncthreads();
            for (int m = rank; m < ntok; m += C) {
                const int64_t src = source(m);
                const uint32_t top = __reduce_max_sync(0xffffffffu, s_max[m][lane & (kR_Warps - 1)]);
                const float amax = __uint_as_float(top);
                int8_t* q = xs + m * p.ks;
                for (int i = K + tid; i < 64 * units; i += kR_Threads) q[i] = 0;
                if (src < 0 || top == 0u || top >= 0x7F800000u) {
                    for (int i = tid; i < K; i += kR_Threads) q[i] = 0;
                    if (tid == 0) s_scale[m] = top >= 0x7F800000u ? __uint_as_float(0x7FC00000u) : 0.0f;
                    continue;
                }
                const typename E::T* x = reinterpret_cast<const typename E::T*>(p.x) + src * p.ldx;
                if (!RowScale::wide(amax)) {
                    const float scale = fmaxf(amax / 127.0f, 1.17549435e-38f);
#pragma unroll 1
                    for (int i = tid; i < K; i += kR_Threads) q[i] = (int8_t)__float2int_rn(E::one(x + i) / scale);
                    if (tid == 0) s_scale[m] = scale;
                    continue;
                }
                const RowScale s(amax);
                for (int i = tid; i < nv; i += kR_Threads) {
                    const typename E::Raw w = E::load8(x + 8 * i);
                    uint2 o;
                    o.x = s.q4(E::value(w, 0), E::value(w, 1), E::value(w, 2), E::value(w, 3));
                    o.y = s.q4(E::value(w, 4), E::value(w, 5), E::value(w, 6), E::value(w, 7));
                    *reinterpret_cast<uint2*>(q + 8 * i) = o;
                }
                for (int i = 8 * nv + tid; i < K; i += kR_Threads) q[i] = (int8_t)s.q(E::one(x + i));
                if (tid == 0) s_scale[m] = s.scale;
            }
            if (C > 1) {   // the others' tokens from their shared memory
                cluster_sync();
                for (int i = tid; i < ntok * 4 * units; i += kR_Threads) {
                    const int m = i / (4 * units), at = m * p.ks + 16 * (i - m * 4 * units), owner = m & (C - 1);
                    if (owner == rank) continue;
                    uint32_t w[4];
                    asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];"
                                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(cluster_addr(smem_u32(xs + at), owner)) : "memory");
                    *reinterpret_cast<uint4*>(xs + at) = make_uint4(w[0], w[1], w[2], w[3]);
                }
                if (tid < ntok && (tid & (C - 1)) != rank) s_scale[tid] = __int_as_float(ld_cluster(cluster_addr(smem_u32(&s_scale[tid]), tid & (C - 1))));
                asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");   // (a CTA's tokens stay until all have read them: the wait is at the end)
            }
        }
        __syncthreads();

        int acc[TILES][4] = {};
        for (int base = 0; base < units; base += kw * kR_Units) {
            if (base > 0 || c0 > start) load(base);
#pragma unroll
            for (int u = 0; u < kR_Units; ++u) {
                const int unit = base + wk + kw * u;
                uint4 x = make_uint4(0, 0, 0, 0);
                if (unit < units && g < ntok) x = *reinterpret_cast<const uint4*>(xs + g * p.ks + 64 * unit + 16 * t);
#pragma unroll
                for (int i = 0; i < TILES; ++i) {
                    const uint4 a = v[u][i][0], b = v[u][i][1];
                    mma_16832(acc[i], a.x, b.x, a.y, b.y, x.x, x.y);
                    mma_16832(acc[i], a.z, b.z, a.w, b.w, x.z, x.w);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < TILES; ++i) {
            red[warp][i][g][2 * t] = acc[i][0];
            red[warp][i][g][2 * t + 1] = acc[i][1];
            red[warp][i][g + 8][2 * t] = acc[i][2];
            red[warp][i][g + 8][2 * t + 1] = acc[i][3];
        }
        __syncthreads();
        for (int o = tid; o < outs * ntok; o += kR_Threads) {   // neighbouring threads: neighbouring outputs of a token
            const int m = o / outs, c = o % outs, n = n0 + c;
            if (n >= mp.N) continue;
            int sum = 0, up = 0;
            for (int w = c / 16 * kw; w < (c / 16 + 1) * kw; ++w) {
                sum += red[w][0][c & 15][m];
                if (DUAL) up += red[w][TILES - 1][c & 15][m];
            }
            float y[2];
            finish2<DUAL>(mp, ch, s_scale[m], 0.0f, sum, 0, up, 0, y);
            const int64_t r = s_row[m];
            if (r >= 0 && r < mp.y_rows) put(mp, r * mp.ldy + n, y[0]);
        }
        __syncthreads();
    }
    if (C > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ---- many tokens ----
constexpr int kW_Tokens = 256, kW_Cols = 256;                 // of a pair's tile: tokens, weight rows (SwiGLU: 128 gate, 128 up)
constexpr int kW_Stage = 2 * kMM_ABytes, kW_Stages = 6;
constexpr int kW_EpiWarps = 16, kW_Threads = 32 * (kMM_FirstEpi + kW_EpiWarps);   // (rows off the 32-byte boundaries with eight: 777 x 4099 of 2000 19.5 us, now 14.6)
// a warp's 32 x 32 results on their way to rows that are not aligned: rows an odd number of words apart
template <int TYPE> __host__ __device__ constexpr int turn_pitch() { return TYPE == kF32 ? 33 : 34; }
template <int TYPE> __host__ __device__ constexpr int turn_bytes() { return 32 * turn_pitch<TYPE>() * (TYPE == kF32 ? 4 : 2); }
template <int TYPE> __host__ __device__ constexpr int turned_stages() { return TYPE == kF32 ? 4 : 5; }
template <int TYPE> __host__ __device__ constexpr int wide_smem(bool vec) {
    return 1024 + (vec ? kW_Stages * kW_Stage : turned_stages<TYPE>() * kW_Stage + kW_EpiWarps * turn_bytes<TYPE>());
}

struct WideShared {
    uint64_t full[kW_Stages], empty[kW_Stages];
    uint64_t tfull[2], tempty[2];
    uint64_t drain;
    uint32_t tmem_base;
    int failed;
    float sw[2][kW_Cols], bias[2][kW_Cols];
};

__device__ __forceinline__ void ld32(uint32_t taddr, int (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
          "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]),
          "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]),
          "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr) : "memory");
}
__device__ __forceinline__ void stg256(void* p, const uint32_t* v) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                 ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}
template <int TYPE>
__device__ __forceinline__ void pack32(const float (&o)[32], uint32_t (&w)[16]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        if (TYPE == kF16) {
            const __half2 h = __floats2half2_rn(o[2 * i], o[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
            const __nv_bfloat162 h = __floats2bfloat162_rn(o[2 * i], o[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
    }
}
// 32 results of one row, all of them inside it and 32-byte aligned
template <int TYPE>
__device__ __forceinline__ void store_row32(typename Out<TYPE>::T* y, const float (&o)[32]) {
    if constexpr (TYPE == kF32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) stg256(y + 8 * i, reinterpret_cast<const uint32_t*>(o) + 8 * i);
    } else {
        uint32_t w[16];
        pack32<TYPE>(o, w);
        stg256(y, w);
        stg256(y + 16, w + 8);
    }
}
// A warp's 32 rows x 32 results from column n on.  r: this lane's row of y, -1 if it has none.
template <int TYPE>
__device__ __forceinline__ void store_block(const MatmulParams& p, typename Out<TYPE>::T* turn, int r, int n, const float (&o)[32], int lane) {
    using T = typename Out<TYPE>::T;
    T* y = reinterpret_cast<T*>(p.y);
    if (p.vec) {
        if (r >= 0) {
            if (n + 32 <= p.N) store_row32<TYPE>(y + r * p.ldy + n, o);
            else {
#pragma unroll
                for (int j = 0; j < 32; ++j) if (n + j < p.N) y[r * p.ldy + n + j] = Out<TYPE>::of(o[j]);
            }
        }
        return;
    }
    // a lane per column: 32 neighbours of a row at a time
    __syncwarp();
    T* mine = turn + lane * turn_pitch<TYPE>();
    if constexpr (TYPE == kF32) {
#pragma unroll
        for (int j = 0; j < 32; ++j) mine[j] = o[j];
    } else {
        uint32_t w[16];
        pack32<TYPE>(o, w);
#pragma unroll
        for (int j = 0; j < 16; ++j) reinterpret_cast<uint32_t*>(mine)[j] = w[j];
    }
    __syncwarp();
    const bool in = n + lane < p.N;
#pragma unroll 8
    for (int i = 0; i < 32; ++i) {
        const int ri = __shfl_sync(0xffffffffu, r, i);
        if (ri >= 0 && in) y[ri * p.ldy + n + lane] = turn[i * turn_pitch<TYPE>() + lane];
    }
}

template <int TYPE, bool DUAL>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kW_Threads, 1) wide_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, MatmulParams p) {
    constexpr int kOuts = DUAL ? 128 : 256;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) WideShared sh;
    __shared__ GroupTable table;
    uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const int rank = blockIdx.x & 1, first = blockIdx.x >> 1, step = gridDim.x >> 1;
    const uint32_t stages = smem_u32(smem);

    if (tid == 0) { prefetch_map(&map_w); prefetch_map(&map_x); }
    if (!p.early) griddep_wait();
    const int total = (p.offsets ? group_table<kW_Tokens, kW_Threads>(p, table) : p.mt) * p.nt;
    if (first >= total) {   // (both CTAs; nothing has been allocated)
        griddep_launch();
        griddep_wait();   // (whoever waits for this grid has what lies before it as well)
        return;
    }
    if (tid == 0) {
        for (int i = 0; i < p.n_stages; ++i) { mbar_init(&sh.full[i], 1); mbar_init(&sh.empty[i], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&sh.tfull[i], 1); mbar_init(&sh.tempty[i], 2 * kW_EpiWarps); }
        mbar_init(&sh.drain, 1);
        sh.failed = 0;
        mbar_fence_init();
    }
    if (warp == 1) tmem_alloc<2>(&sh.tmem_base, 512);
    fence_before();
    __syncthreads();
    cluster_sync();   // the pair's barriers stand before a copy or an MMA reaches over
    fence_after();
    const uint32_t tmem = sh.tmem_base;
    if (tid == 0) griddep_launch();
    const int nkb = (p.K + kMM_KBytes - 1) / kMM_KBytes;

    if (warp == 0) {
        int st = 0;
        uint32_t ph = 0, used = 0;
        bool ok = true, waited = !p.early;
        for (int id = first; ok && id < total; id += step) {
            const Tile t = take_tile<kW_Tokens, kOuts>(p, table, id);
            const bool mine = t.ntok > 128 * rank;   // (a tile of up to 128 tokens is the first CTA's)
            const uint32_t bytes = (t.ntok > 128 ? 4 : 3) * kMM_ABytes;
            const int wrow = DUAL ? rank * p.N + t.n0 : t.n0 + 128 * rank;
            for (int kb = 0; kb < nkb; ++kb) {
                if (!mbar_wait(&sh.empty[st], ph ^ 1u)) { ok = false; break; }
                const uint32_t dst = stages + st * kW_Stage, bar = bar_addr<2>(&sh.full[st]);
                if (elect1()) {
                    if (rank == 0) mbar_expect_tx(&sh.full[st], bytes);   // (both CTAs' copies)
                    tma_3d<2>(dst + kMM_ABytes, &map_w, kb * kMM_KBytes, wrow, t.expert, bar);
                }
                __syncwarp();
                if (!waited) { griddep_wait(); waited = true; }
                if (mine && elect1()) tma_2d<2>(dst, &map_x, kb * kMM_KBytes, t.row0 + 128 * rank, bar);
                __syncwarp();
                used |= 1u << st;
                if (++st == p.n_stages) { st = 0; ph ^= 1u; }
            }
        }
        if (!ok) {   // the copies under way, which the first CTA's barriers count, land before the pair goes
            sh.failed = 1;
            if (rank == 0)
                for (int i = 0; i < p.n_stages; ++i)
                    if (used >> i & 1u) mbar_wait(&sh.full[i], (i < st ? ph : ph ^ 1u));
        }
    } else if (warp == 1 && rank == 0) {
        constexpr uint32_t idesc = idesc_i8(2 * 128, kW_Cols);
        int st = 0, n = 0;
        uint32_t ph = 0;
        bool ok = true;
        for (int id = first; ok && id < total; id += step, ++n) {
            const int buf = n & 1;
            if (!mbar_wait(&sh.tempty[buf], ((n >> 1) & 1) ^ 1u)) { ok = false; break; }
            fence_after();
            const uint32_t d = tmem + buf * kW_Cols;
            for (int kb = 0; kb < nkb; ++kb) {
                if (!mbar_wait(&sh.full[st], ph)) { ok = false; break; }
                fence_after();
                if (elect1()) {
                    const uint32_t a = stages + st * kW_Stage, b = a + kMM_ABytes;
#pragma unroll
                    for (int k = 0; k < kMM_KBytes / 32; ++k) mma_i8<2>(d, desc_sw128(a + 32 * k), desc_sw128(b + 32 * k), idesc, kb > 0 || k > 0);
                    commit<2>(&sh.empty[st]);
                }
                __syncwarp();
                if (++st == p.n_stages) { st = 0; ph ^= 1u; }
            }
            if (ok && elect1()) commit<2>(&sh.tfull[buf]);
            __syncwarp();
        }
        if (!ok) {
            sh.failed = 1;
            if (elect1()) commit<2>(&sh.drain);   // (the MMAs under way)
            __syncwarp();
            mbar_wait(&sh.drain, 0);
        }
    } else if (warp >= kMM_FirstEpi) {
        const int q = warp & 3, part = (warp - kMM_FirstEpi) >> 2, row = q * 32 + lane, et = tid - 32 * kMM_FirstEpi;
        const uint32_t taddr = tmem + ((uint32_t)(q * 32) << 16);
        constexpr int kMine = kOuts / (kW_EpiWarps / 4);   // columns of a warp
        auto* turn = reinterpret_cast<typename Out<TYPE>::T*>(smem + turned_stages<TYPE>() * kW_Stage + (warp - kMM_FirstEpi) * turn_bytes<TYPE>());   // (where rows are not aligned)
        bool ok = true;
        griddep_wait();   // (the tokens' scales; and nothing of y is written before what used its memory has ended)
        // a tile's scales and places are looked up while the one before is on its way
        Tile t;
        float sw_next = 0.0f, bias_next = 0.0f, sx_next;
        int64_t r_next;
        auto look_up = [&](int id) {
            t = take_tile<kW_Tokens, kOuts>(p, table, id);
            if (et < kW_Cols) {
                const int c = DUAL ? t.n0 + (et & 127) : t.n0 + et;   // accumulator column `et`
                const int64_t at = ((int64_t)t.expert * (DUAL ? 2 : 1) + (DUAL ? et >> 7 : 0)) * p.N + c;
                sw_next = c < p.N ? p.sw[at] : 0.0f;
                bias_next = c < p.N && p.bias ? p.bias[at] : 0.0f;
            }
            const int i = 128 * rank + row;   // this thread's token of the tile
            r_next = -1;
            sx_next = 0.0f;
            if (i < t.ntok) {
                sx_next = p.sx[t.row0 + i];
                r_next = p.out_rows ? p.out_rows[t.row0 + i] : t.row0 + i;
            }
        };
        look_up(first);
        int n = 0;
        for (int id = first; id < total; id += step, ++n) {
            const int buf = n & 1, ntok = t.ntok, n0 = t.n0;
            if (et < kW_Cols) { sh.sw[buf][et] = sw_next; sh.bias[buf][et] = bias_next; }
            const int r = r_next >= 0 && r_next < p.y_rows ? (int)r_next : -1;
            float sx = sx_next;
            asm volatile("bar.sync 1, %0;" ::"n"(32 * kW_EpiWarps) : "memory");
            if (id + step < total) look_up(id + step);
            if (ok && !mbar_wait(&sh.tfull[buf], (n >> 1) & 1)) { ok = false; sh.failed = 1; }
            fence_after();
            if (!ok) sx = __uint_as_float(0x7FC00000u);
            if (128 * rank + q * 32 < ntok) {
#pragma unroll 1
                for (int c0 = part * kMine; c0 < (part + 1) * kMine; c0 += 32) {
                    if (n0 + c0 >= p.N) break;
                    int v[32];
                    float o[32];
                    ld32(taddr + buf * kW_Cols + c0, v);
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        const float4 s = *reinterpret_cast<const float4*>(&sh.sw[buf][c0 + j]), b = *reinterpret_cast<const float4*>(&sh.bias[buf][c0 + j]);
                        o[j] = scaled(v[j], s.x, sx, b.x); o[j + 1] = scaled(v[j + 1], s.y, sx, b.y);
                        o[j + 2] = scaled(v[j + 2], s.z, sx, b.z); o[j + 3] = scaled(v[j + 3], s.w, sx, b.w);
                    }
                    if (DUAL) {
                        ld32(taddr + buf * kW_Cols + 128 + c0, v);
#pragma unroll
                        for (int j = 0; j < 32; j += 4) {
                            const float4 s = *reinterpret_cast<const float4*>(&sh.sw[buf][128 + c0 + j]), b = *reinterpret_cast<const float4*>(&sh.bias[buf][128 + c0 + j]);
                            float y[2];
                            silu_mul2(o[j], o[j + 1], scaled(v[j], s.x, sx, b.x), scaled(v[j + 1], s.y, sx, b.y), y);
                            o[j] = y[0]; o[j + 1] = y[1];
                            silu_mul2(o[j + 2], o[j + 3], scaled(v[j + 2], s.z, sx, b.z), scaled(v[j + 3], s.w, sx, b.w), y);
                            o[j + 2] = y[0]; o[j + 3] = y[1];
                        }
                    } else if (p.act == CHIMERE_ACT_RELU2) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) o[j] = relu2(o[j]);
                    }
                    store_block<TYPE>(p, turn, r, n0 + c0, o, lane);
                }
            }
            fence_before();
            __syncwarp();
            if (lane == 0) arrive_cluster(cluster_addr(smem_u32(&sh.tempty[buf]), 0));
        }
    }
    fence_before();
    __syncthreads();
    cluster_sync();   // nothing of the other CTA's reaches over any more
    fence_after();
    if (warp == 1) tmem_free<2>(tmem, 512);
    if (tid == 0 && sh.failed && p.status) atomicOr(p.status, kStatusWaitTimeout);
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                              CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encoder() {
    static EncodeFn fn = nullptr;   // (the same address whoever looks it up first)
    if (!fn) {
        void* at = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &at, 12000, cudaEnableDefault, &found) == cudaSuccess && found == cudaDriverEntryPointSuccess)
            fn = (EncodeFn)at;
        else cudaGetLastError();
    }
    return fn;
}
// rows of K bytes as boxes of 128 bytes x box_rows
bool make_map(CUtensorMap* map, const void* base, int K, int64_t rows, int64_t planes, int64_t ld, int64_t plane, int box_rows, int rank) {
    const cuuint64_t dims[3] = {(cuuint64_t)K, (cuuint64_t)rows, (cuuint64_t)planes};
    const cuuint64_t strides[2] = {(cuuint64_t)ld, (cuuint64_t)plane};
    const cuuint32_t box[3] = {kMM_KBytes, (cuuint32_t)box_rows, 1}, one[3] = {1, 1, 1};
    return encoder()(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, rank, const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct MatmulCall {
    const int8_t* x;
    int64_t ldx;
    const int8_t* w;
    int64_t ldw, w_plane;
    MatmulParams p;
    bool dual;
};

cudaLaunchConfig_t launch_config(int grid, size_t smem, int cluster, bool pdl, cudaStream_t stream, cudaLaunchAttribute (&attr)[2]) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(kMM_Threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    int n = 0;
    if (pdl) { attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization; attr[n++].val.programmaticStreamSerializationAllowed = 1; }
    if (cluster > 1) { attr[n].id = cudaLaunchAttributeClusterDimension; attr[n].val.clusterDim.x = cluster; attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1; ++n; }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    return cfg;
}

template <int BN, bool DUAL>
int launch_tile(const MatmulCall& c, int tiles, int split, bool pdl, cudaStream_t stream) {
    constexpr int kStage = kMM_ABytes * (DUAL ? 2 : 1) + BN * kMM_KBytes;
    static bool done[64];
    CUtensorMap mx, mw;
    MatmulParams p = c.p;
    if (!make_map(&mx, c.x, p.K, p.M, 1, c.ldx, 0, BN, 2)) return -5;
    if (!make_map(&mw, c.w, p.K, (DUAL ? 2 : 1) * (int64_t)p.N, p.E, c.ldw, c.w_plane, 128, 3)) return -5;
    const int nkb = (p.K + kMM_KBytes - 1) / kMM_KBytes, most = (200 * 1024) / kStage;
    int stages = (nkb + split - 1) / split;
    const int parts = split > 1 ? (BN * (DUAL ? 2 : 1) * 512 + kStage - 1) / kStage : 1;   // room for the sums
    stages = stages < parts ? parts : stages;
    if (split == 1 && stages < most) stages = most;
    stages = stages > most ? most : stages;
    stages = stages > kMM_MaxStages ? kMM_MaxStages : stages;
    p.n_stages = stages;
    p.split = split;
    p.mt = (p.M + BN - 1) / BN;
    p.nt = (p.N + 127) / 128;
    auto kernel = matmul_kernel<BN, DUAL>;
    cudaError_t e = max_smem_once(kernel, 1024 + 200 * 1024, done);
    if (e != cudaSuccess) return -(100 + (int)e);
    const int grid = split > 1 ? tiles * split : tiles < sm_count() ? tiles : sm_count();
    cudaLaunchAttribute attr[2];
    const cudaLaunchConfig_t cfg = launch_config(grid, 1024 + (size_t)stages * kStage, split, pdl, stream, attr);
    e = cudaLaunchKernelEx(&cfg, kernel, mx, mw, p);
    return e == cudaSuccess ? 0 : -(100 + (int)e);
}

template <int TYPE, bool DUAL>
int launch_wide(const MatmulCall& c, int64_t tiles, bool pdl, cudaStream_t stream) {
    static bool done[64];
    CUtensorMap mx, mw;
    MatmulParams p = c.p;
    if (!make_map(&mx, c.x, p.K, p.M, 1, c.ldx, 0, 128, 2)) return -5;
    if (!make_map(&mw, c.w, p.K, (DUAL ? 2 : 1) * (int64_t)p.N, p.E, c.ldw, c.w_plane, 128, 3)) return -5;
    constexpr int kOuts = DUAL ? 128 : 256, kSize = TYPE == kF32 ? 4 : 2;
    p.mt = (p.M + kW_Tokens - 1) / kW_Tokens;
    p.nt = (p.N + kOuts - 1) / kOuts;
    p.split = 1;
    p.vec = ((uintptr_t)p.y & 31) == 0 && p.ldy * kSize % 32 == 0;
    p.n_stages = p.vec ? kW_Stages : turned_stages<TYPE>();
    auto kernel = wide_kernel<TYPE, DUAL>;
    constexpr int kMost = wide_smem<TYPE>(true) > wide_smem<TYPE>(false) ? wide_smem<TYPE>(true) : wide_smem<TYPE>(false);
    static_assert(kMost + (int)sizeof(WideShared) + (int)sizeof(GroupTable) <= 227 * 1024, "one CTA's shared memory");
    cudaError_t e = max_smem_once(kernel, kMost, done);
    if (e != cudaSuccess) return -(100 + (int)e);
    const int pairs = sm_count() / 2;
    cudaLaunchAttribute attr[2];
    cudaLaunchConfig_t cfg = launch_config(2 * (int)(tiles < pairs ? tiles : pairs), wide_smem<TYPE>(p.vec), 1, pdl, stream, attr);
    cfg.blockDim = dim3(kW_Threads);
    e = cudaLaunchKernelEx(&cfg, kernel, mx, mw, p);
    return e == cudaSuccess ? 0 : -(100 + (int)e);
}

// Token tiles of width bn: of a dense call exactly, of a grouped one at most.
int64_t token_tiles(const MatmulCall& c, int bn) {
    return c.p.offsets ? c.p.M / bn + (c.p.M < c.p.E ? c.p.M : c.p.E) : (c.p.M + bn - 1) / bn;
}

// warps of a CTA that share K: as many as have kR_Units units each
int rows_warps(int K) {
    int kw = 1;
    while (kw < kR_Warps && kw * kR_Units * 64 < K) kw *= 2;
    return kw;
}
int rows_outs(int K) { return 16 * (kR_Warps / rows_warps(K)); }

template <int TYPE, bool DUAL>
int launch_rows(const MatmulCall& c, const QuantParams* x, bool pdl, cudaStream_t stream) {
    static bool done[64];
    RowsParams r{};
    r.m = c.p;
    r.x = x ? x->x : c.x;
    r.ldx = x ? x->ldx : c.ldx;
    if (x) { r.x_rows = x->x_rows; r.rows = x->rows; r.rows_div = x->rows_div; r.vec = x->vec; }
    r.w = c.w; r.ldw = c.ldw; r.w_plane = c.w_plane;
    const int units = (c.p.K + 63) / 64, tokens = c.p.M < kR_Tokens ? c.p.M : kR_Tokens;
    r.ks = 64 * (units | 1);
    r.kw = rows_warps(c.p.K);
    const int outs = rows_outs(c.p.K);
    r.cluster = 1;
    while (!c.p.offsets && TYPE != kI8 && r.cluster < c.p.M) r.cluster *= 2;
    auto kernel = rows_kernel<TYPE, DUAL>;
    cudaError_t e = max_smem_once(kernel, kR_Tokens * 64 * (kR_MaxK / 64 + 1), done);
    if (e != cudaSuccess) return -(100 + (int)e);
    cudaLaunchAttribute attr[2];
    const int ctas = (c.p.N + outs - 1) / outs;
    cudaLaunchConfig_t cfg = launch_config((ctas + r.cluster - 1) / r.cluster * r.cluster, (size_t)tokens * r.ks, r.cluster, pdl, stream, attr);
    cfg.blockDim = dim3(kR_Threads);
    cfg.gridDim.y = c.p.offsets ? c.p.M : 1;
    e = cudaLaunchKernelEx(&cfg, kernel, r);
    return e == cudaSuccess ? 0 : -(100 + (int)e);
}
template <int TYPE>
int launch_rows_type(const MatmulCall& c, const QuantParams* x, bool pdl, cudaStream_t stream) {
    return c.dual ? launch_rows<TYPE, true>(c, x, pdl, stream) : launch_rows<TYPE, false>(c, x, pdl, stream);
}
// x null: rows that are quantised already
int launch_rows_any(const MatmulCall& c, const QuantParams* x, int x_type, bool pdl, cudaStream_t stream) {
    if (!x) return launch_rows_type<kI8>(c, x, pdl, stream);
    return x_type == kF32 ? launch_rows_type<kF32>(c, x, pdl, stream) : x_type == kF16 ? launch_rows_type<kF16>(c, x, pdl, stream) : launch_rows_type<kBF16>(c, x, pdl, stream);
}
// Batches for the kernel of a few tokens: dense ones of up to four (4096 x 2048, us, this / tensor-core tiles: 1 token 4.4 / 6.1, 4: 5.1 / 6.1, 6: 5.9 / 6.1; 2048 x
// 4096 6: 6.9 / 6.9; 4096 x 8192 3: 11.9 / 11.9, 6: 17.3 / 12.1).  Grouped ones while their CTAs, if every pair has a group of its own, are four per SM at most (experts of 512 x 2048,
// both products, 8 pairs 12.3 / 18.4, 16: 20.5 / 20.5, 32: 34 / 27; of 1856 x 2688 6 pairs, 696 and 1008 CTAs, 24.6 / 20.6; of 2048 x 2048 4 pairs 21 / 25, 8: 31 / 26), and no more than 32 pairs, since they may all be one group's, which
// its CTAs take eight at a time.
constexpr int kR_DenseTokens = 4, kR_MaxCtas = 4 * 148, kR_MaxPairs = 32;
bool few_tokens(const MatmulCall& c) {
    if (c.p.K > kR_MaxK) return false;
    return c.p.offsets ? c.p.M <= kR_MaxPairs && (int64_t)c.p.M * ((c.p.N + rows_outs(c.p.K) - 1) / rows_outs(c.p.K)) <= kR_MaxCtas : c.p.M <= kR_DenseTokens;
}
// ... whose CTAs quantise the tokens themselves, in clusters: dense ones of up to eight tokens, rows of up to 2048 values (one token: up to kR_MaxK) and two CTAs per SM.  us,
// in one launch / with one in front: 1024 x 2048 1 token 3.8 / 4.6, 8: 6.1 / 7.2; 4096 x 2048 1: 4.9 / 4.6, 4: 6.4 / 6.1, 8: 7.4 / 7.4; 512 x 512 8: 5.4 / 6.1; 2048 x 4096 1: 5.9 / 6.1,
// 8: 11.0 / 8.5; 3712 x 2688 7: 9.4 / 7.7; 8192 x 4096 (512 CTAs) 1: 12.4 / 9.4; 16384 x 2048 8: 23 / 12.
constexpr int kR_InlineK = 2048;
bool few_values(int64_t M, int N, int K) { return M <= kR_Tokens && K <= (M == 1 ? kR_MaxK : kR_InlineK) && (N + rows_outs(K) - 1) / rows_outs(K) <= 2 * 148; }
bool few_values(const MatmulCall& c) { return c.p.offsets ? few_tokens(c) : few_values(c.p.M, c.p.N, c.p.K); }

int launch_matmul(const MatmulCall& c, bool pdl, cudaStream_t stream) {
    if (c.p.M == 0) return 0;
    if (few_tokens(c)) return launch_rows_any(c, nullptr, 0, pdl, stream);
    if (!encoder()) return -6;
    const int sms = sm_count();
    // Pairs of CTAs: dense batches of more than 128 tokens with sixteen tiles or more, grouped ones of 32 tokens per group or more on average.  us, by pairs / by single CTAs:
    //   dense    4096 x 2048 (16 tiles up to 256 tokens) 128 tokens 11.1 / 9.0, 192: 11.0 / 11.1, 384: 11.4 / 14.5; 8192 x 4096 (32) 128: 16.0 / 14.3, 192: 15.8 / 20.4;
    //            2048 x 4096 256 tokens (8) 15.5 / 10.6, 384 (16) 15.6 / 14.1; 2048 x 2048 384 (16) 11.1 / 11.1
    //   grouped  gate and up + down of experts of 512 x 2048.  256 groups, even: 16 tokens each 176 / 143, 32: 188 / 163, 48: 187 / 187, 64: 192 / 241; with Zipf routing (some 30
    //            groups in use) 16: 38 / 64, 32: 56 / 92, 64: 79 / 163.  64 even groups of 16: 53 / 43, 32: 55 / 50, 64: 59 / 64.  4 groups of 32: 19.7 / 16.9, 64: 20.7 / 20.4,
    //            128: 22.4 / 21.9; 16 of 32: 22.1 / 21.9, 128: 26.2 / 33.9.  128 even groups of 1856 x 2688, 32 each: 263 / 218, 64: 269 / 248.
    //            The average does not see how the rows are spread: the line lies between what even and skewed routing would ask for.
    const int outs = c.dual ? 128 : 256;
    const int64_t wide = token_tiles(c, kW_Tokens) * ((c.p.N + outs - 1) / outs);
    if (c.p.offsets ? c.p.M >= 32 * (int64_t)c.p.E : c.p.M > 128 && wide >= 16) {
        if (wide > 0x3FFFFFFF) return -2;
        switch (c.p.y_type) {
            case kF32: return c.dual ? launch_wide<kF32, true>(c, wide, pdl, stream) : launch_wide<kF32, false>(c, wide, pdl, stream);
            case kF16: return c.dual ? launch_wide<kF16, true>(c, wide, pdl, stream) : launch_wide<kF16, false>(c, wide, pdl, stream);
            default: return c.dual ? launch_wide<kBF16, true>(c, wide, pdl, stream) : launch_wide<kBF16, false>(c, wide, pdl, stream);
        }
    }
    // Width of the token tiles and the CTAs that share one.
    const int64_t nt = (c.p.N + 127) / 128;
    const int nkb = (c.p.K + kMM_KBytes - 1) / kMM_KBytes;
    int bn = 16, split = 1;
    if (c.p.offsets) {
        bn = c.p.M < c.p.E ? 16 : c.p.M < 4 * (int64_t)c.p.E ? 32 : 64;
        while (split < 8 && token_tiles(c, bn) * nt * split * 2 <= sms && split * 4 <= nkb) split *= 2;
    } else {
        // cycles: a stage is its bytes through L2 (50 per cycle); a tile's results, and with a shared tile the exchange of its parts
        double best = 1e30;
        for (int b = 16; b <= 64; b *= 2) {
            const int64_t tiles = (int64_t)(c.p.M + b - 1) / b * nt;
            const int tokens = c.p.M < b ? c.p.M : b;
            for (int s = 1; s <= 8 && (s == 1 || (tiles * s <= sms && s * 2 <= nkb)); s *= 2) {
                const double stage = (16384.0 * (c.dual ? 2 : 1) + 128.0 * b) / 50.0, tail = s > 1 ? 1200.0 + 20.0 * tokens : 25.0 * tokens;
                const double cost = (double)((tiles * s + sms - 1) / sms) * ((nkb + s - 1) / s * stage + tail);
                if (cost < best) { best = cost; bn = b; split = s; }
            }
        }
    }
    const int64_t tiles = token_tiles(c, bn) * nt;
    if (tiles > 0x3FFFFFFF) return -2;
    switch (bn + (c.dual ? 1 : 0)) {
        case 16: return launch_tile<16, false>(c, (int)tiles, split, pdl, stream);
        case 32: return launch_tile<32, false>(c, (int)tiles, split, pdl, stream);
        case 64: return launch_tile<64, false>(c, (int)tiles, split, pdl, stream);
        case 17: return launch_tile<16, true>(c, (int)tiles, split, pdl, stream);
        case 33: return launch_tile<32, true>(c, (int)tiles, split, pdl, stream);
        default: return launch_tile<64, true>(c, (int)tiles, split, pdl, stream);
    }
}

// A batch's pairs share rows: from so many values on each row is quantised once and copied to its pairs (32768 pairs of 2048 values, eight per row, bf16: 37 us when each pair
// quantises its own, 9 + 16 so).
constexpr int64_t kGatherValues = 1 << 22;
bool gather_apart(int64_t pairs, int top_k, int K) { return top_k > 1 && pairs * K >= kGatherValues; }

// Rows of f32, f16 or bf16 times a matrix: quantised in the product's own CTAs where that is little, else by a kernel in front.  `first`: nothing of this
// call has been launched before.
// `apart` (with x.rows): scratch for the x_rows rows of x and their scales, quantised once and copied; null: each row of the product quantises its own.
int launch_linear(MatmulCall c, QuantParams x, int x_type, bool first, int8_t* apart, float* apart_scale, cudaStream_t stream) {
    x.vec = ((uintptr_t)x.x & 15) == 0 && (x.ldx * (x_type == kF32 ? 4 : 2)) % 16 == 0;
    c.p.early = !first;
    if (few_values(c)) return launch_rows_any(c, &x, x_type, !first, stream);
    if (!x.q || !x.scale) return -4;      // (what is left needs room for the quantised rows)
    if (!few_tokens(c) && !encoder()) return -6;
    QuantParams once = x;
    if (apart) { once.rows = nullptr; once.rows_div = 1; once.M = x.x_rows; once.q = apart; once.scale = apart_scale; }
    cudaError_t e = launch_quantize(once, x_type, stream, !first);
    if (e == cudaSuccess && apart)
        e = launch_pdl(gather_rows_kernel, dim3((unsigned)((x.M + 7) / 8)), 256, 0, stream, (const int8_t*)apart, (const float*)apart_scale, x.x_rows, x.rows, x.rows_div, x.q, x.scale, x.M,
                       x.ldq);
    if (e != cudaSuccess) return -(100 + (int)e);
    c.p.early = true;
    return launch_matmul(c, true, stream);
}

// ------------------------------------------------------------------ checks ----
inline bool float_type(int t) { return t == kF32 || t == kF16 || t == kBF16; }
inline int type_size(int t) { return t == kF32 ? 4 : 2; }
inline bool misaligned(const void* p, int to) { return ((uintptr_t)p & (uintptr_t)(to - 1)) != 0; }

// (one_launch: the quantised rows and their scales stay in the product's CTAs, q and scale are null)
int check_quantize(const void* x, int type, int64_t ldx, int64_t x_rows, const int32_t* rows, int rows_div, int64_t M, int K, const int8_t* q, int64_t ldq, const float* scale,
                   bool one_launch = false) {
    if (M < 0 || M > 0x7FFFFFFF || x_rows < 0 || K <= 0 || K > kMaxK || ldx < K || ldq < K || ldq % 16 || rows_div <= 0) return -2;
    if (!float_type(type)) return -3;
    if (!rows && x_rows < M) return -2;
    if (M == 0) return 0;
    if ((!x && x_rows > 0) || (!one_launch && (!q || !scale))) return -1;
    if (misaligned(x, type_size(type)) || misaligned(q, 16) || misaligned(scale, 4) || misaligned(rows, 4)) return -5;
    return 0;
}
int check_matmul(const int8_t* x, int64_t ldx, const float* sx, const int8_t* w, int64_t ldw, int64_t w_plane, const float* sw, const float* bias, int E, int64_t M, int N, int K,
                 int act, const void* y, int y_type, int64_t ldy, int64_t y_rows, const int32_t* out_rows, bool one_launch = false) {
    const int64_t R = (act == CHIMERE_ACT_SWIGLU ? 2 : 1) * (int64_t)N;
    if (M < 0 || M > kMaxRows || N <= 0 || R > 0x7FFFFF00 || K <= 0 || K > kMaxK || E <= 0 || E > kMaxGroups) return -2;
    if (ldx < K || ldw < K || ldx % 16 || ldw % 16 || ldy < N || y_rows < 0) return -2;
    if (E > 1 && (w_plane % 16 || w_plane < (R - 1) * ldw + K)) return -2;
    if (act != CHIMERE_ACT_NONE && act != CHIMERE_ACT_SWIGLU && act != CHIMERE_ACT_RELU2) return -2;
    if (!float_type(y_type)) return -3;
    if (!out_rows && y_rows < M) return -2;
    if (M == 0) return 0;
    if ((!one_launch && (!x || !sx)) || !w || !sw || (!y && y_rows > 0)) return -1;
    if (misaligned(x, 16) || misaligned(w, 16) || misaligned(sx, 4) || misaligned(sw, 4) || misaligned(bias, 4) || misaligned(y, type_size(y_type)) || misaligned(out_rows, 4)) return -5;
    return 0;
}
// Rows of `bytes` bytes each, `pitch` apart.  Two matrices share memory if their ranges do, but for such with one pitch that lie side by side.
struct RowsRange { uintptr_t at; int64_t pitch, bytes, rows; };
bool share_memory(const RowsRange& a, const RowsRange& b) {
    if (a.rows == 0 || b.rows == 0) return false;
    const uintptr_t a_end = a.at + (uintptr_t)(a.pitch * (a.rows - 1) + a.bytes), b_end = b.at + (uintptr_t)(b.pitch * (b.rows - 1) + b.bytes);
    if (a_end <= b.at || b_end <= a.at) return false;
    if (a.rows == 1 || b.rows == 1 || a.pitch != b.pitch) return true;
    const RowsRange &lo = a.at <= b.at ? a : b, &hi = a.at <= b.at ? b : a;
    const int64_t off = (int64_t)((hi.at - lo.at) % (uintptr_t)a.pitch);
    return off < lo.bytes || off + hi.bytes > a.pitch;
}
MatmulCall matmul_call(const int8_t* x, int64_t ldx, const float* sx, const int8_t* w, int64_t ldw, int64_t w_plane, const float* sw, const float* bias, const int32_t* offsets, int E,
                       int64_t M, int N, int K, int act, void* y, int y_type, int64_t ldy, int64_t y_rows, const int32_t* out_rows, int32_t* status, bool early) {
    MatmulCall c{};
    c.x = x; c.ldx = ldx; c.w = w; c.ldw = ldw;
    c.dual = act == CHIMERE_ACT_SWIGLU;
    c.w_plane = E > 1 ? w_plane : (c.dual ? 2 : 1) * (int64_t)N * ldw;
    MatmulParams& p = c.p;
    p.sx = sx; p.sw = sw; p.bias = bias; p.y = y; p.ldy = ldy; p.y_rows = y_rows; p.offsets = offsets; p.out_rows = out_rows; p.status = status;
    p.M = (int)M; p.N = N; p.K = K; p.E = E; p.y_type = y_type; p.act = act; p.early = early;
    return c;
}
inline int up16(int k) { return (k + 15) & ~15; }
inline int up8(int k) { return (k + 7) & ~7; }
inline size_t up256(size_t v) { return (v + 255) & ~(size_t)255; }
inline size_t rows_bytes(int64_t M, int K) { return up256((size_t)M * up16(K)) + up256((size_t)M * 4); }   // int8 rows and their scales
struct Carver {
    uint8_t* base;
    size_t at;
    void* take(size_t n) { void* r = (void*)((uintptr_t)base + at); at += up256(n); return r; }
};
inline int rc_of(cudaError_t e) { return e == cudaSuccess ? 0 : -(100 + (int)e); }

}  // namespace
}  // namespace chimere

using namespace chimere;

extern "C" {

int chimere_b200_quantize_i8(const void* d_x, int x_type, int64_t ldx, int64_t x_rows, const int32_t* d_rows, int rows_div, int64_t M, int K,
                             int8_t* d_q, int64_t ldq, float* d_scale, cudaStream_t stream) {
    const int rc = check_quantize(d_x, x_type, ldx, x_rows, d_rows, rows_div, M, K, d_q, ldq, d_scale);
    if (rc || M == 0) return rc;
    return rc_of(launch_quantize(QuantParams{d_x, ldx, x_rows, d_rows, rows_div, K, d_q, ldq, d_scale, M, 0}, x_type, stream, false));
}

int chimere_b200_matmul_w8a8(const int8_t* d_x, int64_t ldx, const float* d_x_scale, const int8_t* d_w, int64_t ldw, const float* d_w_scale, const float* d_bias,
                             int64_t M, int N, int K, int act, void* d_y, int y_type, int64_t ldy, int32_t* d_status, cudaStream_t stream) {
    const int rc = check_matmul(d_x, ldx, d_x_scale, d_w, ldw, 0, d_w_scale, d_bias, 1, M, N, K, act, d_y, y_type, ldy, M, nullptr);
    if (rc || M == 0) return rc;
    return launch_matmul(matmul_call(d_x, ldx, d_x_scale, d_w, ldw, 0, d_w_scale, d_bias, nullptr, 1, M, N, K, act, d_y, y_type, ldy, M, nullptr, d_status, false), false, stream);
}

int chimere_b200_matmul_w8a8_grouped(const int8_t* d_x, int64_t ldx, const float* d_x_scale, const int8_t* d_w, int64_t ldw, int64_t stride_w, const float* d_w_scale,
                                     const float* d_bias, const int32_t* d_offsets, int E, int64_t M, int N, int K, int act, void* d_y, int y_type, int64_t ldy,
                                     int64_t y_rows, const int32_t* d_out_rows, int32_t* d_status, cudaStream_t stream) {
    const int rc = check_matmul(d_x, ldx, d_x_scale, d_w, ldw, stride_w, d_w_scale, d_bias, E, M, N, K, act, d_y, y_type, ldy, y_rows, d_out_rows);
    if (rc || M == 0) return rc;
    if (!d_offsets) return -1;
    if (misaligned(d_offsets, 4)) return -5;
    return launch_matmul(matmul_call(d_x, ldx, d_x_scale, d_w, ldw, stride_w, d_w_scale, d_bias, d_offsets, E, M, N, K, act, d_y, y_type, ldy, y_rows, d_out_rows, d_status, false), false, stream);
}

int64_t chimere_b200_linear_w8a8_bytes(int64_t M, int N, int K) {
    if (M < 0 || M > kMaxRows || N <= 0 || K <= 0 || K > kMaxK) return -2;
    return M == 0 || few_values(M, N, K) ? 0 : (int64_t)rows_bytes(M, K);
}

int chimere_b200_linear_w8a8(const void* d_x, int x_type, int64_t ldx, const int8_t* d_w, int64_t ldw, const float* d_w_scale, const float* d_bias, int64_t M, int N, int K,
                             int act, void* d_y, int y_type, int64_t ldy, void* d_ws, size_t ws_bytes, int32_t* d_status, cudaStream_t stream) {
    const bool one_launch = few_values(M, N, K);
    const int64_t rows = M < 0 ? 0 : M;
    Carver ws{(uint8_t*)d_ws, 0};
    int8_t* q = one_launch ? nullptr : (int8_t*)ws.take((size_t)rows * up16(K));
    float* scale = one_launch ? nullptr : (float*)ws.take((size_t)rows * 4);
    if (M > 0 && !one_launch && !d_ws) return -1;
    if (misaligned(d_ws, 256)) return -5;
    int rc = check_quantize(d_x, x_type, ldx, M, nullptr, 1, M, K, q, up16(K), scale, one_launch);
    if (rc) return rc;
    rc = check_matmul(q, up16(K), scale, d_w, ldw, 0, d_w_scale, d_bias, 1, M, N, K, act, d_y, y_type, ldy, M, nullptr, one_launch);
    if (rc || M == 0) return rc;
    if (ws_bytes < ws.at) return -4;
    // in one launch some CTAs still read x when others store y
    const int x_size = type_size(x_type), y_size = type_size(y_type);
    if (one_launch && share_memory({(uintptr_t)d_x, ldx * x_size, (int64_t)K * x_size, M}, {(uintptr_t)d_y, ldy * y_size, (int64_t)N * y_size, M})) return -2;
    return launch_linear(matmul_call(q, up16(K), scale, d_w, ldw, 0, d_w_scale, d_bias, nullptr, 1, M, N, K, act, d_y, y_type, ldy, M, nullptr, d_status, false),
                         QuantParams{d_x, ldx, M, nullptr, 1, K, q, up16(K), scale, M, 0}, x_type, true, nullptr, nullptr, stream);
}

int64_t chimere_b200_experts_w8a8_bytes(int64_t T, int top_k, int H, int F) {
    if (T < 0 || top_k <= 0 || T > kMaxRows / top_k || H <= 0 || F <= 0 || H > kMaxK || F > kMaxK) return -2;
    const int64_t pairs = T * top_k;
    return (int64_t)(rows_bytes(pairs, H) + rows_bytes(pairs, F) + up256((size_t)pairs * up8(F) * 4) + (gather_apart(pairs, top_k, H) ? rows_bytes(T, H) : 0));
}

int chimere_b200_experts_w8a8(const void* d_x, int x_type, int64_t ldx, int64_t T, const int32_t* d_perm, const int32_t* d_offsets, int top_k, int E,
                              const int8_t* d_w_up, int64_t ld_up, int64_t stride_up, const float* d_up_scale,
                              const int8_t* d_w_down, int64_t ld_down, int64_t stride_down, const float* d_down_scale,
                              int H, int F, int act, void* d_y, int y_type, int64_t ldy, void* d_ws, size_t ws_bytes, int32_t* d_status, cudaStream_t stream) {
    if (T < 0 || top_k <= 0 || T > kMaxRows / top_k) return -2;
    if (H <= 0 || F <= 0 || H > kMaxK || F > kMaxK) return -2;
    if (act != CHIMERE_ACT_SWIGLU && act != CHIMERE_ACT_RELU2) return -2;
    const int64_t P = T * top_k;
    Carver ws{(uint8_t*)d_ws, 0};
    int8_t* q = (int8_t*)ws.take((size_t)P * up16(H));
    float* scale = (float*)ws.take((size_t)P * 4);
    int8_t* hq = (int8_t*)ws.take((size_t)P * up16(F));
    float* h_scale = (float*)ws.take((size_t)P * 4);
    float* h = (float*)ws.take((size_t)P * up8(F) * 4);
    int8_t* apart = nullptr;
    float* apart_scale = nullptr;
    if (gather_apart(P, top_k, H)) {
        apart = (int8_t*)ws.take((size_t)T * up16(H));
        apart_scale = (float*)ws.take((size_t)T * 4);
    }
    if (P > 0 && (!d_ws || !d_perm || !d_offsets)) return -1;
    if (misaligned(d_ws, 256) || misaligned(d_offsets, 4)) return -5;
    int rc = check_quantize(d_x, x_type, ldx, T, d_perm, top_k, P, H, q, up16(H), scale);
    if (rc) return rc;
    rc = check_matmul(q, up16(H), scale, d_w_up, ld_up, stride_up, d_up_scale, nullptr, E, P, F, H, act, h, kF32, up8(F), P, nullptr);
    if (rc) return rc;
    rc = check_matmul(hq, up16(F), h_scale, d_w_down, ld_down, stride_down, d_down_scale, nullptr, E, P, H, F, CHIMERE_ACT_NONE, d_y, y_type, ldy, P, d_perm);
    if (rc || P == 0) return rc;
    if (ws_bytes < ws.at) return -4;
    rc = launch_linear(matmul_call(q, up16(H), scale, d_w_up, ld_up, stride_up, d_up_scale, nullptr, d_offsets, E, P, F, H, act, h, kF32, up8(F), P, nullptr, d_status, false),
                       QuantParams{d_x, ldx, T, d_perm, top_k, H, q, up16(H), scale, P, 0}, x_type, true, apart, apart_scale, stream);
    if (rc) return rc;
    return launch_linear(matmul_call(hq, up16(F), h_scale, d_w_down, ld_down, stride_down, d_down_scale, nullptr, d_offsets, E, P, H, F, CHIMERE_ACT_NONE, d_y, y_type, ldy, P, d_perm,
                                     d_status, false),
                         QuantParams{h, up8(F), P, nullptr, 1, F, hq, up16(F), h_scale, P, 0}, kF32, false, nullptr, nullptr, stream);
}

}  // extern "C"
