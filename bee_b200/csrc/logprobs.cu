// Log probabilities of given tokens under logits / T, with the entropy of each
// row's distribution and its k most likely alternatives, and the gradient.
//
// None of these exist in the reference.  Per row of `vocab` logits x, with
// m = max x, z_i = (x_i - m) / T, S = sum e^{z_i}:
//   logp_i = z_i - log S            H = log S - (sum e^{z_i} z_i) / S
//   dx_i   = (gl (delta_{i,target} - p_i) - gH p_i (logp_i + H)) / T
// Forward reads the logits once (one exponential an element), backward reads
// and writes them once: both are bound by HBM.
//
// One pass: every thread keeps its own running maximum m, S and
// Z = sum e^{z} z (in units of log2), and rescales them when its maximum grows;
// the (m, S, Z) triples are joined over the block, in a fixed order, at the end.
// All statistics are fp32.  x - m is formed before the scaling, so that the
// error of z does not grow with the size of the logits.
//
// Alternatives: the stream keeps, per thread, the maxima of its two best batches
// of chunks, which they are, and the best of the others.  The maxima of 64 groups of
// threads (the same lane of half of the warps) give a bound: the k-th largest of them
// is reached by an element of each of k groups, so it is at most the k-th largest
// element, and on rows without structure only about 64 ln(64 / (64 - k)) elements
// reach it (24 for k = 20, 44 for k = 32).  Each warp reads the batches of its threads whose
// maxima do again (one or two of a thread, all of them if its third may), an element
// per lane, and lists the elements that reach the bound; the rank of each among all is
// counted.  Order is that of (value, ~index) keys of 64 bits: ties go to the lowest index.
// Where fewer than k elements are unmasked, masked ones follow by index.  Rows with more
// elements that reach the bound than a list holds (many ties) insert them one by one into
// sorted lists instead.
// This costs latency at the end of a row (4 rows of 131072 bf16: 4.5 us without
// alternatives, 8.3 us with 20); sorting the group maxima and merging the warps' lists
// took 1 to 4 us more, reading the whole shares of the threads concerned 2 to 10 us.
//
// Few rows: a cluster of up to 8 CTAs shares a row and joins its partial
// results through distributed shared memory (no workspace, fixed order).
#include <cmath>

#include "common.cuh"
#include "sm100.cuh"

namespace bee_b200 {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kTopMax = 32;
// Floor of z * log2(e): 2^-16384 is 0 in fp32, and 0 * -16384 is 0, so masked
// (-inf) and far-off logits add nothing to S and Z; a NaN passes through.
constexpr float kZFloor = -16384.f;
// How far (in powers of two) a term may exceed 1 before the sums are moved to the
// new maximum: 2^30 terms of 2^16 stay far inside fp32.
constexpr float kSlack = 16.f;

__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ float ex2(float x) {
    float d;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(d) : "f"(x));
    return d;
}

// 16-byte chunks of logits as floats.  The maxima ignore NaNs (they reach S).
template <typename T> struct Elems;
template <> struct Elems<float> {
    static constexpr int E = 4;
    static __device__ __forceinline__ float get(const float* p) { return *p; }
    static __device__ __forceinline__ void put(float* p, float v) { *p = v; }
    static __device__ __forceinline__ void unpack(uint4 q, float* v) {
        v[0] = __uint_as_float(q.x); v[1] = __uint_as_float(q.y); v[2] = __uint_as_float(q.z); v[3] = __uint_as_float(q.w);
    }
    static __device__ __forceinline__ uint4 pack(const float* v) {
        return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    }
    static __device__ __forceinline__ float max(uint4 q) {
        return fmaxf(fmaxf(__uint_as_float(q.x), __uint_as_float(q.y)), fmaxf(__uint_as_float(q.z), __uint_as_float(q.w)));
    }
    template <int N> static __device__ __forceinline__ float max(const uint4 (&q)[N]) {
        float m = max(q[0]);
#pragma unroll
        for (int j = 1; j < N; ++j) m = fmaxf(m, max(q[j]));
        return m;
    }
    static __device__ __forceinline__ uint4 fill() { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }
};
template <> struct Elems<__nv_bfloat16> {
    static constexpr int E = 8;
    static __device__ __forceinline__ float get(const __nv_bfloat16* p) { return __bfloat162float(*p); }
    static __device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
    static __device__ __forceinline__ void unpack(uint4 q, float* v) {
        v[0] = bf16_lo(q.x); v[1] = bf16_hi(q.x); v[2] = bf16_lo(q.y); v[3] = bf16_hi(q.y);
        v[4] = bf16_lo(q.z); v[5] = bf16_hi(q.z); v[6] = bf16_lo(q.w); v[7] = bf16_hi(q.w);
    }
    static __device__ __forceinline__ uint4 pack(const float* v) {
        return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
    }
    static __device__ __forceinline__ __nv_bfloat162 h2(uint32_t w) { return *reinterpret_cast<__nv_bfloat162*>(&w); }
    static __device__ __forceinline__ __nv_bfloat162 max2(uint4 q) { return __hmax2(__hmax2(h2(q.x), h2(q.y)), __hmax2(h2(q.z), h2(q.w))); }
    template <int N> static __device__ __forceinline__ float max(const uint4 (&q)[N]) {
        __nv_bfloat162 m = max2(q[0]);
#pragma unroll
        for (int j = 1; j < N; ++j) m = __hmax2(m, max2(q[j]));
        const float2 f = __bfloat1622float2(m);
        return fmaxf(f.x, f.y);
    }
    static __device__ __forceinline__ float max(uint4 q) {
        const float2 f = __bfloat1622float2(max2(q));
        return fmaxf(f.x, f.y);
    }
    static __device__ __forceinline__ uint4 fill() { return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u); }
};
template <> struct Elems<__half> {
    static constexpr int E = 8;
    static __device__ __forceinline__ float get(const __half* p) { return __half2float(*p); }
    static __device__ __forceinline__ void put(__half* p, float v) { *p = __float2half_rn(v); }
    static __device__ __forceinline__ __half2 h2(uint32_t w) { return *reinterpret_cast<__half2*>(&w); }
    static __device__ __forceinline__ void unpack(uint4 q, float* v) {
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(h2(w[i]));
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
    static __device__ __forceinline__ uint4 pack(const float* v) {
        return make_uint4(pack_f16x2(v[0], v[1]), pack_f16x2(v[2], v[3]), pack_f16x2(v[4], v[5]), pack_f16x2(v[6], v[7]));
    }
    static __device__ __forceinline__ __half2 max2(uint4 q) { return __hmax2(__hmax2(h2(q.x), h2(q.y)), __hmax2(h2(q.z), h2(q.w))); }
    template <int N> static __device__ __forceinline__ float max(const uint4 (&q)[N]) {
        __half2 m = max2(q[0]);
#pragma unroll
        for (int j = 1; j < N; ++j) m = __hmax2(m, max2(q[j]));
        const float2 f = __half22float2(m);
        return fmaxf(f.x, f.y);
    }
    static __device__ __forceinline__ float max(uint4 q) {
        const float2 f = __half22float2(max2(q));
        return fmaxf(f.x, f.y);
    }
    static __device__ __forceinline__ uint4 fill() { return make_uint4(0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u); }
};

// A row as 16-byte aligned chunks, whatever its own alignment: chunk c holds
// elements [c*E - lead, c*E - lead + E) of the row, where `lead` elements of
// its first 16 bytes lie before it.  Chunks wholly inside the row are one
// vector load; the first and last may be partial and are read element by
// element (nothing outside the row is touched), absent elements as -inf.
template <typename T> struct RowChunks {
    static constexpr int E = Elems<T>::E;
    const T* row;
    const uint4* base;
    int lead, chunks, full_lo, full_hi;  // chunks in [full_lo, full_hi) are whole
    long long n;
    __device__ __forceinline__ RowChunks(const T* r, long long vocab) : row(r), n(vocab) {
        lead = static_cast<int>((reinterpret_cast<uintptr_t>(r) & 15u) / sizeof(T));
        base = reinterpret_cast<const uint4*>(r - lead);
        chunks = static_cast<int>((lead + vocab + E - 1) / E);
        full_lo = lead ? 1 : 0;
        full_hi = static_cast<int>((lead + vocab) / E);
    }
    __device__ __forceinline__ bool whole(int c) const { return c >= full_lo && c < full_hi; }
    __device__ __forceinline__ long long first(int c) const { return static_cast<long long>(c) * E - lead; }
    __device__ __forceinline__ uint4 partial(int c) const {
        float v[E];
        const long long i0 = first(c);
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = (i0 + e >= 0 && i0 + e < n) ? Elems<T>::get(row + i0 + e) : -INFINITY;
        return Elems<T>::pack(v);  // exact: the values come from this type
    }
    __device__ __forceinline__ uint4 load(int c) const { return whole(c) ? __ldg(base + c) : partial(c); }
};

// ---------------------------------------------------------------- online statistics

struct Stat {
    float m, s, z;  // maximum, sum of 2^(z_i), sum of 2^(z_i) z_i; z_i = (x_i - m) / T * log2(e)
};

// Adds the sums of 2^z and 2^z z over a chunk, z = (x - m) c.  Where x is -inf the
// second would be 0 * -inf = NaN; FLOOR replaces z below kZFloor by it.
template <typename T, bool FLOOR>
__device__ __forceinline__ void chunk_sums(uint4 q, uint64_t negm2, uint64_t c2, uint64_t& s2, uint64_t& z2) {
    constexpr int E = Elems<T>::E;
    float v[E];
    Elems<T>::unpack(q, v);
#pragma unroll
    for (int e = 0; e < E; e += 2) {
        const uint64_t d = mul_f32x2(add_f32x2(pack_f32x2(v[e], v[e + 1]), negm2), c2);
        float lo, hi;
        unpack_f32x2(d, lo, hi);
        if (FLOOR) {
            lo = max_nan(lo, kZFloor);
            hi = max_nan(hi, kZFloor);
        }
        const uint64_t e2 = pack_f32x2(ex2(lo), ex2(hi));
        s2 = add_f32x2(s2, e2);
        z2 = fma_f32x2(e2, FLOOR ? pack_f32x2(lo, hi) : d, z2);
    }
}
__device__ __forceinline__ float pair_sum(uint64_t v) {
    float lo, hi;
    unpack_f32x2(v, lo, hi);
    return lo + hi;
}

__device__ __forceinline__ float finite_max(float m) { return m == -INFINITY ? 0.f : m; }

// Moves the sums from maximum st.m to maximum m (>= st.m).
__device__ __forceinline__ void rebase(Stat& st, float m, float c) {
    if (st.s != 0.f && st.m != m) {  // s is 0 only while the maximum is -inf; a NaN stays
        const float d = fmaxf((st.m - m) * c, kZFloor);
        const float r = ex2(d);
        st.z = r * fmaf(d, st.s, st.z);
        st.s *= r;
    }
    st.m = m;
}

// The warp's statistics, in every lane: one maximum, then each lane's sums moved to it and added.
__device__ __forceinline__ Stat warp_join(Stat st, float c) {
    rebase(st, warp_max(st.m), c);
    st.s = warp_sum(st.s);
    st.z = warp_sum(st.z);
    return st;
}

// ---------------------------------------------------------------- keys

// Order of fp32 values as unsigned integers (-0 equals +0).
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t b = __float_as_uint(v + 0.f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float from_ordered(uint32_t o) {
    return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
__device__ __forceinline__ uint64_t make_key(float v, uint32_t index) {
    return (static_cast<uint64_t>(ordered(v)) << 32) | static_cast<uint32_t>(~index);
}

// One step of a bitonic merge over the lanes: the lane keeps the larger value
// of itself and lane ^ d if `up`, else the smaller.
template <typename K> __device__ __forceinline__ K exchange(K k, int d, bool up) {
    const K o = __shfl_xor_sync(0xffffffffu, k, d);
    return ((o > k) == up) ? o : k;
}
// The 32 largest of a list sorted largest first and `other`, the other list's value at 31 - lane.
template <typename K> __device__ __forceinline__ K merge_lanes(K k, K other, int lane) {
    k = other > k ? other : k;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) k = exchange(k, d, (lane & d) == 0);
    return k;
}

// ---------------------------------------------------------------- forward

struct LogprobArgs {
    const void* logits;
    const void* targets;
    int targets_i64;
    long long ld, rows, vocab;
    float inv_t;
    int top;
    float *logprob, *entropy, *row_max, *log_sum, *top_logprobs;
    int* top_ids;
};

__device__ __forceinline__ long long target_of(const void* t, int is64, long long r) {
    return is64 ? static_cast<const long long*>(t)[r] : static_cast<const int*>(t)[r];
}

constexpr int kUnroll = 4;  // chunks of a thread per batch
constexpr int kStages = 3;  // batches in its part of the shared-memory ring
// CTAs that may share a row.  A row of a 128-thread block has at most 513 chunks, for which cluster_for never
// gains from more than 4.
constexpr int max_cluster(int threads) { return threads == 128 ? 4 : 8; }

// 16 bytes from global to shared memory, both addresses moved by OFF bytes.
template <int OFF> __device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0 + %2], [%1 + %2], 16;" ::"r"(dst), "l"(src), "n"(OFF) : "memory");
}
template <int OFF> __device__ __forceinline__ uint4 lds16(uint32_t src) {
    uint4 q;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4 + %5];" : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w) : "r"(src), "n"(OFF) : "memory");
    return q;
}

// One CTA's part of a row: the whole chunks [lo, hi) and perhaps the partial
// first or last chunk of the row.
template <typename T> struct Part {
    RowChunks<T> row;
    int lo, hi, edge_lo, edge_hi;  // edge_lo, edge_hi: index of the partial chunk, or -1
    __device__ __forceinline__ Part(const LogprobArgs& a, long long r, int rank, int cluster)
        : row(static_cast<const T*>(a.logits) + r * a.ld, a.vocab) {
        const int whole = max(row.full_hi - row.full_lo, 0), per = (whole + cluster - 1) / cluster;
        lo = row.full_lo + min(whole, rank * per);
        hi = row.full_lo + min(whole, (rank + 1) * per);
        edge_lo = rank == 0 && row.full_lo > 0 ? 0 : -1;
        edge_hi = rank == cluster - 1 && row.full_hi < row.chunks && row.full_hi >= row.full_lo ? row.full_hi : -1;
    }
};

// A forward CTA's shared memory beside its ring.
template <int THREADS, bool TOP> struct ForwardShared {
    static constexpr int WARPS = THREADS / 32, CLUSTER = max_cluster(THREADS);
    Stat warp_stat[WARPS];
    Stat cta_stat[CLUSTER];  // rank 0's copy is filled by the whole cluster
    // for the alternatives:
    alignas(16) float group_max[TOP ? 64 : 4];
    float lane_max[TOP ? WARPS : 1][32];
    uint64_t lists[TOP ? WARPS : 1][32];  // each warp's elements that reach the bound
    uint64_t sorted[TOP ? 32 : 1];
    uint64_t cta_list[TOP ? CLUSTER : 1][32];
    int listed[WARPS];

    static constexpr int RING = sizeof(uint4) * kStages * kUnroll * THREADS;
};

// Clusters of `cluster` CTAs (1: single CTAs) take rows in grid-stride order.
// Every thread streams its own chunks of the coming batches, across rows, into
// its own slots of a ring with cp.async, so that loads stay in flight while a row
// is joined and its alternatives are sought; no barrier is needed for the ring.
template <typename T, int THREADS, bool TOP>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) token_logprobs_kernel(const LogprobArgs a, int cluster) {
    constexpr int WARPS = THREADS / 32;
    constexpr int E = Elems<T>::E;
    using Shared = ForwardShared<THREADS, TOP>;
    // The grid is made for 1024 threads per SM: a CTA that found no place would wait for all the rows of another.  (An
    // SM has 228 KiB, and each CTA takes 1 KiB beside its own.)
    static_assert((sizeof(Shared) + Shared::RING + 1024) * (1024 / THREADS) <= 228 * 1024, "fewer CTAs fit an SM than the grid is made for");
    extern __shared__ __align__(16) uint4 ring[];  // [kStages][kUnroll][THREADS]
    __shared__ Shared sh;
    auto& warp_stat = sh.warp_stat;
    auto& cta_stat = sh.cta_stat;
    auto& group_max = sh.group_max;
    auto& lane_max = sh.lane_max;
    auto& lists = sh.lists;
    auto& cta_list = sh.cta_list;
    auto& sorted = sh.sorted;
    auto& listed = sh.listed;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = cluster > 1 ? static_cast<int>(sm100::cluster_ctarank()) : 0;
    const float c = a.inv_t * kLog2e;
    if (cluster > 1) sm100::cluster_sync();  // every CTA of the cluster runs before its shared memory is written
    pdl_wait();
    const long long step = gridDim.x / cluster, r0 = blockIdx.x / cluster;

    static_assert(kUnroll == 4, "the four chunks of a batch are written out");
    constexpr int STEP = THREADS * 16, SLOT = kUnroll * STEP;  // bytes between a thread's chunks; a slot of the ring
    const uint32_t ring_lo = sm100::smem_u32(ring) + tid * 16, ring_hi = ring_lo + kStages * SLOT;
    // the batch to copy next: this thread's first chunk of it, the whole batches and chunks left in the part, its slot
    long long issue_row = r0;
    const uint4* issue_from = nullptr;
    int issue_whole = 0, issue_rest = 0;
    uint32_t issue_to = ring_lo;
    auto open_row = [&] {
        if (issue_row >= a.rows) return;
        const Part<T> p(a, issue_row, rank, cluster);
        issue_from = p.row.base + p.lo + tid;
        issue_whole = (p.hi - p.lo) / (kUnroll * THREADS);
        issue_rest = (p.hi - p.lo) % (kUnroll * THREADS);
    };
    auto issue = [&] {
        if (issue_whole > 0) {
            cp_async16<0>(issue_to, issue_from);
            cp_async16<STEP>(issue_to, issue_from);
            cp_async16<2 * STEP>(issue_to, issue_from);
            cp_async16<3 * STEP>(issue_to, issue_from);
            issue_from += kUnroll * THREADS;
            --issue_whole;
        } else if (issue_rest > 0) {
            const int left = issue_rest - tid;
            if (left > 0) cp_async16<0>(issue_to, issue_from);
            if (left > THREADS) cp_async16<STEP>(issue_to, issue_from);
            if (left > 2 * THREADS) cp_async16<2 * STEP>(issue_to, issue_from);
            if (left > 3 * THREADS) cp_async16<3 * STEP>(issue_to, issue_from);
            issue_rest = 0;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");  // empty past the end: the wait counts stay uniform
        issue_to = issue_to + SLOT == ring_hi ? ring_lo : issue_to + SLOT;
        while (issue_whole == 0 && issue_rest == 0 && issue_row < a.rows) {  // on to the next row that has whole chunks
            issue_row += step;
            open_row();
        }
    };
    open_row();
    while (issue_whole == 0 && issue_rest == 0 && issue_row < a.rows) {
        issue_row += step;
        open_row();
    }
    for (int j = 1; j < kStages; ++j) issue();

    uint32_t slot = ring_lo;
    // targets are read a row ahead, by the thread that writes the row's results, so that nothing waits for them
    const bool writer = tid == 0 && rank == 0 && a.logprob;
    long long next_target = writer && r0 < a.rows ? target_of(a.targets, a.targets_i64, r0) : -1;
    for (long long r = r0; r < a.rows; r += step) {
        if (r + step >= a.rows) pdl_trigger();  // this CTA's last row
        const Part<T> part(a, r, rank, cluster);
        const RowChunks<T>& row = part.row;

        // early loads: the target's logit and the partial chunks
        const long long target = next_target;
        float xt = 0.f;
        if (writer) {
            xt = target < 0 ? 0.f : target < a.vocab ? Elems<T>::get(row.row + target) : NAN;
            if (r + step < a.rows) next_target = target_of(a.targets, a.targets_i64, r + step);
        }
        const int edge = tid == 0 ? part.edge_lo : tid == 1 ? part.edge_hi : -1;
        uint4 edge_chunk = Elems<T>::fill();
        if (edge >= 0) edge_chunk = row.partial(edge);

        Stat st{-INFINITY, 0.f, 0.f};  // st.m: a reference, at most kSlack below the maximum, so that it seldom moves
        // the maximum; TOP: also those of this thread's two best batches, their numbers, and the best of the rest
        float top = -INFINITY, m1 = -INFINITY, m2 = -INFINITY, m3 = -INFINITY;
        int b1 = 0, b2 = 0;
        bool floored = false;  // this thread has met logits so low that z or 2^z z overflows
        auto consume = [&](uint4 (&q)[kUnroll], int b) {  // b: the batch's number, -1 for the partial chunks
            const float bm = Elems<T>::max(q);
            top = fmaxf(top, bm);
            if (TOP && b >= 0) {
                const bool first = bm > m1, second = bm > m2;
                m3 = second ? m2 : fmaxf(m3, bm);
                m2 = first ? m1 : second ? bm : m2;
                b2 = first ? b1 : second ? b : b2;
                m1 = first ? bm : m1;
                b1 = first ? b : b1;
            }
            if ((bm - st.m) * c > kSlack) rebase(st, bm, c);
            const float m = finite_max(st.m);
            const uint64_t negm2 = pack_f32x2(-m, -m), c2 = pack_f32x2(c, c);
            uint64_t s2 = 0, z2 = 0;  // pairs of fp32 zeros
            if (!floored) {
#pragma unroll
                for (int j = 0; j < kUnroll; ++j) chunk_sums<T, false>(q[j], negm2, c2, s2, z2);
                floored = pair_sum(z2) != pair_sum(z2);
            }
            if (floored) {  // -inf, or a NaN
                s2 = z2 = 0;
#pragma unroll 1
                for (int j = 0; j < kUnroll; ++j) {
                    chunk_sums<T, true>(q[0], negm2, c2, s2, z2);
                    q[0] = q[1];
                    q[1] = q[2];
                    q[2] = q[3];
                }
            }
            st.s += pair_sum(s2);
            st.z += pair_sum(z2);
        };
        // whole batches, then one for the chunks that are left, then the row's partial chunks
        const int whole = (part.hi - part.lo) / (kUnroll * THREADS), rest = (part.hi - part.lo) % (kUnroll * THREADS);
        const uint4 none = Elems<T>::fill();
        for (int b = 0; b < whole; ++b) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
            issue();
            uint4 q[kUnroll] = {lds16<0>(slot), lds16<STEP>(slot), lds16<2 * STEP>(slot), lds16<3 * STEP>(slot)};
            slot = slot + SLOT == ring_hi ? ring_lo : slot + SLOT;
            consume(q, b);
        }
        if (rest > 0) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
            issue();
            const int left = rest - tid;  // this thread's chunks are those at 0, THREADS, ... below it
            if (left > 0) {
                uint4 q[kUnroll] = {lds16<0>(slot), left > THREADS ? lds16<STEP>(slot) : none,
                                    left > 2 * THREADS ? lds16<2 * STEP>(slot) : none, left > 3 * THREADS ? lds16<3 * STEP>(slot) : none};
                consume(q, whole);
            }
            slot = slot + SLOT == ring_hi ? ring_lo : slot + SLOT;
        }
        if (edge >= 0) {
            uint4 q[kUnroll] = {edge_chunk, none, none, none};
            consume(q, -1);
        }
        __syncwarp();

        if constexpr (TOP) {
            lane_max[warp][lane] = top;
            if (tid < 32) sorted[tid] = 0;
            __syncthreads();
            // the bound: the smallest group maximum that fewer than k others exceed (every warp finds it for itself;
            // all of them write the same 64 maxima)
            float g0 = lane_max[0][lane], g1 = lane_max[WARPS / 2][lane];
#pragma unroll
            for (int w = 1; w < WARPS / 2; ++w) {
                g0 = fmaxf(g0, lane_max[w][lane]);
                g1 = fmaxf(g1, lane_max[WARPS / 2 + w][lane]);
            }
            group_max[lane] = g0;
            group_max[32 + lane] = g1;
            __syncwarp();
            int n0 = 0, n1 = 0;
#pragma unroll 4
            for (int i = 0; i < 16; ++i) {
                const float4 g = reinterpret_cast<const float4*>(group_max)[i];
                n0 += (g.x > g0) + (g.y > g0) + (g.z > g0) + (g.w > g0);
                n1 += (g.x > g1) + (g.y > g1) + (g.z > g1) + (g.w > g1);
            }
            const uint32_t o0 = n0 < a.top ? ordered(g0) : 0xffffffffu, o1 = n1 < a.top ? ordered(g1) : 0xffffffffu;
            // (where fewer than k groups hold anything unmasked, every unmasked element is a candidate)
            const float bound = fmaxf(from_ordered(__reduce_min_sync(0xffffffffu, o0 < o1 ? o0 : o1)), -3.402823466e+38f);

            // the warp's elements that reach it
            const int batches = whole + (rest > 0);
            int held = 0;
            auto list = [&](float x, long long i) {  // an element per lane, NaN for none
                const uint32_t hit = __ballot_sync(0xffffffffu, x >= bound);
                const int at = held + __popc(hit & ((1u << lane) - 1u));
                if (x >= bound && at < 32) lists[warp][at] = make_key(x, static_cast<uint32_t>(i));
                held += __popc(hit);
            };
            const bool every = m3 >= bound;  // more than two of this thread's batches may reach it
            int b = every ? 0 : b1, todo = every ? batches : static_cast<int>(m1 >= bound) + static_cast<int>(m2 >= bound);
            constexpr int AHEAD = 4;  // batches whose loads are in flight together
            const int chunk = lane / E;  // this lane's element of a batch: element lane % E of its owner's chunk lane / E
#pragma unroll 1
            for (uint32_t left = __ballot_sync(0xffffffffu, todo > 0); left != 0 && held <= 32; left = __ballot_sync(0xffffffffu, todo > 0)) {
                const int mine = part.lo + b * kUnroll * THREADS + tid;
                float x[AHEAD];
                long long at[AHEAD];
                uint32_t now = left;
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) {
                    const int from = now ? __ffs(now) - 1 : 0;
                    const int cc = __shfl_sync(0xffffffffu, mine, from) + chunk * THREADS;
                    at[i] = row.first(cc) + lane % E;
                    x[i] = now != 0 && chunk < kUnroll && cc < part.hi ? Elems<T>::get(row.row + at[i]) : NAN;
                    now &= now - 1;  // 0 stays 0
                }
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) list(x[i], at[i]);
                if ((left & ~now) >> lane & 1u) {
                    --todo;
                    b = every ? b + 1 : b2;
                }
            }
            if (warp == 0) {  // the partial chunks
                float x[2] = {NAN, NAN};
                long long at[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int e = i == 0 ? part.edge_lo : part.edge_hi;
                    at[i] = row.first(e) + lane;
                    if (e >= 0 && lane < E && at[i] >= 0 && at[i] < row.n) x[i] = Elems<T>::get(row.row + at[i]);
                }
                list(x[0], at[0]);
                list(x[1], at[1]);
            }
            if (lane == 0) listed[warp] = held;
            if (lane >= held) lists[warp][lane] = 0;
            __syncthreads();
            int longest = 0, found = 0;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                longest = max(longest, listed[w]);
                found += listed[w];
            }
            if (longest <= 32) {
                // fewer than k unmasked elements: masked ones follow by index, and fewer than k of the first 64 are not masked
                if (warp == 0 && found < a.top) {
                    const long long i0 = part.edge_lo >= 0 ? 0 : row.first(part.lo);
                    const long long i1 = part.edge_hi >= 0 ? row.n : min(row.n, row.first(part.hi));
                    int place = found;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const long long i = i0 + h * 32 + lane;
                        const bool masked = i < i1 && Elems<T>::get(row.row + i) == -INFINITY;
                        const uint32_t all = __ballot_sync(0xffffffffu, masked);
                        const int at = place + __popc(all & ((1u << lane) - 1u));
                        if (masked && at < a.top) sorted[at] = make_key(-INFINITY, static_cast<uint32_t>(i));
                        place += __popc(all);
                    }
                }
                if (lane < held) {
                    const uint64_t key = lists[warp][lane];
                    int place = 0;  // the keys above this one; the lists' ends are 0
#pragma unroll 2
                    for (int i = 0; i < longest; ++i)
#pragma unroll
                        for (int w = 0; w < WARPS; ++w) place += lists[w][i] > key;
                    if (place < a.top) sorted[place] = key;
                }
            } else {
                // inserts the elements of each lane's chunk (index cc, none where !in) that reach the bound into the
                // warp's sorted list: chunk by chunk, its elements spread over the lanes
                uint64_t best = 0;
                auto insert = [&](uint4 q0, int cc, bool in) {
                    const float cm = Elems<T>::max(q0);
                    // no key of the chunk is larger than this one
                    const uint64_t most = in && cm >= bound ? make_key(cm, static_cast<uint32_t>(max(row.first(cc), 0ll))) : 0;
                    uint32_t hits = __ballot_sync(0xffffffffu, most > __shfl_sync(0xffffffffu, best, a.top - 1));
#pragma unroll 1
                    while (hits) {
                        const int from = __ffs(hits) - 1;
                        hits &= hits - 1;
                        if (__shfl_sync(0xffffffffu, most, from) <= __shfl_sync(0xffffffffu, best, a.top - 1)) continue;
                        const long long i = row.first(__shfl_sync(0xffffffffu, cc, from)) + lane;
                        const float x = lane < E && i >= 0 && i < row.n ? Elems<T>::get(row.row + i) : NAN;
                        const uint64_t ck = x >= bound ? make_key(x, static_cast<uint32_t>(i)) : 0;
                        uint32_t more = __ballot_sync(0xffffffffu, ck > __shfl_sync(0xffffffffu, best, a.top - 1));
#pragma unroll 1
                        while (more) {
                            const int src = __ffs(more) - 1;
                            more &= more - 1;
                            const uint64_t nk = __shfl_sync(0xffffffffu, ck, src);
                            const int pos = __popc(__ballot_sync(0xffffffffu, best > nk));
                            const uint64_t up = __shfl_up_sync(0xffffffffu, best, 1);
                            best = lane < pos ? best : lane == pos ? nk : up;
                        }
                    }
                };
#pragma unroll 1
                for (int cb = part.lo + warp * 32; cb < part.hi; cb += THREADS) {
                    const int cc = cb + lane;
                    insert(cc < part.hi ? __ldg(row.base + cc) : none, cc, cc < part.hi);
                }
                insert(edge_chunk, edge, edge >= 0);
                __syncthreads();  // the lists above are no longer read
                lists[warp][lane] = best;
                __syncthreads();
                if (warp == 0) {
#pragma unroll 1
                    for (int w = 1; w < WARPS; ++w) best = merge_lanes(best, lists[w][31 - lane], lane);
                    if (lane < a.top) sorted[lane] = best;
                }
            }
        }

        // join the block's statistics, then the cluster's, each in a fixed order
        rebase(st, top, c);
        st = warp_join(st, c);
        if (lane == 0) warp_stat[warp] = st;
        __syncthreads();
        uint64_t best = 0;  // TOP, warp 0: key of this lane's alternative
        if (warp == 0) {
            st = warp_join(lane < WARPS ? warp_stat[lane] : Stat{-INFINITY, 0.f, 0.f}, c);
            if (TOP) best = sorted[lane];
        }
        if (cluster > 1) {
            if (warp == 0) {
                const uint32_t dst = sm100::mapa_shared(sm100::smem_u32(&cta_stat[rank]), 0);
                if (lane < 3) {
                    const float v = lane == 0 ? st.m : lane == 1 ? st.s : st.z;
                    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst + 4 * lane), "f"(v) : "memory");
                }
                if constexpr (TOP) {
                    const uint32_t dk = sm100::mapa_shared(sm100::smem_u32(&cta_list[rank][lane]), 0);
                    asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(dk), "l"(best) : "memory");
                }
            }
            __syncwarp();
            sm100::cluster_sync();
            if (rank == 0) {
                if (warp == 0) st = warp_join(lane < cluster ? cta_stat[lane] : Stat{-INFINITY, 0.f, 0.f}, c);
                if constexpr (TOP) {
#pragma unroll 1
                    for (int half = cluster / 2; half > 0; half >>= 1) {  // a tree over the CTAs' lists, a warp per pair
                        if (warp < half)
                            cta_list[warp][lane] = merge_lanes(cta_list[warp][lane], cta_list[warp + half][31 - lane], lane);
                        __syncthreads();
                    }
                    best = cta_list[0][lane];
                }
            }
            if (r + step < a.rows) sm100::cluster_sync();  // rank 0 has read the partial results: the next row's may come
        }
        if (warp == 0 && rank == 0) {
            const bool empty = st.m == -INFINITY && st.s == 0.f;
            const float m = finite_max(st.m);
            const float log_s = logf(st.s);  // -inf for an empty row
            if (lane == 0) {
                if (a.logprob)
                    a.logprob[r] = target < 0 ? 0.f : empty ? (target < a.vocab ? -INFINITY : NAN) : (xt - m) * a.inv_t - log_s;
                if (a.entropy) a.entropy[r] = empty ? 0.f : fmaf(-kLn2, st.z / st.s, log_s);
                if (a.row_max) a.row_max[r] = st.m;
                if (a.log_sum) a.log_sum[r] = log_s;
            }
            if constexpr (TOP) {
                if (lane < a.top) {
                    const bool bad = st.s != st.s;  // a NaN or +inf: no distribution
                    const float v = from_ordered(static_cast<uint32_t>(best >> 32));
                    a.top_ids[r * a.top + lane] = bad ? -1 : static_cast<int>(~static_cast<uint32_t>(best));
                    a.top_logprobs[r * a.top + lane] = bad ? NAN : empty ? -INFINITY : (v - m) * a.inv_t - log_s;
                }
            }
        }
        __syncthreads();  // the shared arrays are reused by the next row
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// ---------------------------------------------------------------- backward

struct LogprobGradArgs {
    const void* logits;
    const void* targets;
    int targets_i64;
    long long ld, ldd, rows, vocab;
    float inv_t;
    const float *row_max, *log_sum, *entropy, *dlogprob, *dentropy;
    void* dlogits;
};

// dx_i = p_i (A + B logp_i) + [i == target] gl / T, A = -(gl + gH H) / T, B = -gH / T.
struct RowGrad {
    float m, log2_s, ga, gb, gt, c;
    bool zero;
    long long target;
    __device__ __forceinline__ float operator()(float x, long long i) const {
        const float lp2 = max_nan((x - m) * c, kZFloor) - log2_s;
        return fmaf(ex2(lp2), fmaf(gb, lp2, ga), i == target ? gt : 0.f);
    }
    // the same for a chunk of elements i0, i0 + 1, ...
    template <int E> __device__ __forceinline__ void chunk(float (&v)[E], long long i0) const {
        const uint64_t negm = pack_f32x2(-m, -m), c2 = pack_f32x2(c, c), negs = pack_f32x2(-log2_s, -log2_s);
        const uint64_t a2 = pack_f32x2(ga, ga), b2 = pack_f32x2(gb, gb);
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            float lo, hi;
            unpack_f32x2(mul_f32x2(add_f32x2(pack_f32x2(v[e], v[e + 1]), negm), c2), lo, hi);
            const uint64_t lp = add_f32x2(pack_f32x2(max_nan(lo, kZFloor), max_nan(hi, kZFloor)), negs);
            unpack_f32x2(lp, lo, hi);
            unpack_f32x2(mul_f32x2(pack_f32x2(ex2(lo), ex2(hi)), fma_f32x2(b2, lp, a2)), v[e], v[e + 1]);
        }
        const long long at = target - i0;
        if (at >= 0 && at < E) {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (e == at) v[e] += gt;
        }
    }
};

__device__ __forceinline__ RowGrad row_grad(const LogprobGradArgs& a, long long r) {
    RowGrad g;
    const float m = a.row_max[r];
    g.target = a.dlogprob ? target_of(a.targets, a.targets_i64, r) : -1;
    float gl = g.target >= 0 ? a.dlogprob[r] : 0.f;
    if (g.target >= a.vocab && gl != 0.f) gl = NAN;  // as the forward's logprob
    const float gh = a.dentropy ? a.dentropy[r] : 0.f;
    g.m = m;
    g.c = a.inv_t * kLog2e;
    g.log2_s = a.log_sum[r] * kLog2e;
    g.ga = -a.inv_t * (gl + (gh != 0.f ? gh * a.entropy[r] : 0.f));
    g.gb = -a.inv_t * kLn2 * gh;
    g.gt = a.inv_t * gl;
    g.zero = (gl == 0.f && gh == 0.f) || (m == -INFINITY && a.log_sum[r] == -INFINITY);
    return g;
}

// One CTA takes segments of THREADS * kUnroll chunks.  VEC: logits and
// gradients have the same offset from a 16-byte boundary in every row.
template <typename T, int THREADS, bool VEC>
__global__ void __launch_bounds__(THREADS, 1280 / THREADS) token_logprobs_grad_kernel(const LogprobGradArgs a, long long segments) {
    constexpr int E = Elems<T>::E;
    pdl_wait();
    for (long long item = blockIdx.x; item < a.rows * segments; item += gridDim.x) {
        if (item + gridDim.x >= a.rows * segments) pdl_trigger();
        const long long r = item / segments;
        const int seg = static_cast<int>(item - r * segments);
        const RowGrad g = row_grad(a, r);
        T* drow = static_cast<T*>(a.dlogits) + r * a.ldd;
        const RowChunks<T> row(static_cast<const T*>(a.logits) + r * a.ld, a.vocab);
        const int c0 = seg * THREADS * kUnroll + threadIdx.x;
        if constexpr (VEC) {
            uint4* dbase = reinterpret_cast<uint4*>(drow - row.lead);
            uint4 q[kUnroll];
#pragma unroll
            for (int j = 0; j < kUnroll; ++j) {
                const int cc = c0 + j * THREADS;
                if (!g.zero && row.whole(cc)) q[j] = __ldcs(row.base + cc);
            }
#pragma unroll
            for (int j = 0; j < kUnroll; ++j) {
                const int cc = c0 + j * THREADS;
                if (cc >= row.chunks) break;
                const long long i0 = row.first(cc);
                if (row.whole(cc)) {
                    float v[E];
                    if (g.zero) {
#pragma unroll
                        for (int e = 0; e < E; ++e) v[e] = 0.f;
                    } else {
                        Elems<T>::unpack(q[j], v);
                        g.chunk(v, i0);
                    }
                    __stcs(dbase + cc, Elems<T>::pack(v));
                } else {
                    for (int e = 0; e < E; ++e)
                        if (i0 + e >= 0 && i0 + e < row.n)
                            Elems<T>::put(drow + i0 + e, g.zero ? 0.f : g(Elems<T>::get(row.row + i0 + e), i0 + e));
                }
            }
        } else {
            for (int j = 0; j < kUnroll * E; ++j) {
                const long long i = (static_cast<long long>(seg) * kUnroll * E + j) * THREADS + threadIdx.x;
                if (i < a.vocab) Elems<T>::put(drow + i, g.zero ? 0.f : g(Elems<T>::get(row.row + i), i));
            }
        }
    }
}

// ---------------------------------------------------------------- host side

// CTAs that share a row: the cluster size with the least work on the slowest
// CTA, a row costing its share of the chunks plus about 1024 chunks' time for its
// joins, and 128 more for each doubling of the cluster.
int cluster_for(long long rows, long long chunks, long long slots, int most) {
    int best = 1;
    double least = 0, joins = 1024;
    for (int cl = 1; cl <= most; cl *= 2, joins += 128) {
        const long long clusters = slots / cl;
        const double cost = static_cast<double>((rows + clusters - 1) / clusters) * (static_cast<double>(chunks) / cl + joins);
        if (cl == 1 || cost < least) {
            least = cost;
            best = cl;
        }
    }
    return best;
}

template <typename T, int THREADS, bool TOP> int launch_forward(const LogprobArgs& a, cudaStream_t st) {
    const long long chunks = (a.vocab + Elems<T>::E - 1) / Elems<T>::E + 1;
    const long long slots = static_cast<long long>(sm_count()) * (1024 / THREADS);
    const int cl = cluster_for(a.rows, chunks, slots, max_cluster(THREADS));
    const size_t smem = ForwardShared<THREADS, TOP>::RING;
    auto logprobs_kern = token_logprobs_kernel<T, THREADS, TOP>;
    static SmemLimit limit;
    if (int rc = limit.ensure(logprobs_kern, static_cast<int>(smem), "token_logprobs")) return rc;
    const long long most = slots / cl;
    const unsigned grid = static_cast<unsigned>((a.rows < most ? a.rows : most) * cl);
    if (cl > 1) launch_pdl_cluster(logprobs_kern, grid, THREADS, static_cast<unsigned>(cl), smem, st, a, cl);
    else launch_pdl(logprobs_kern, grid, THREADS, smem, st, a, 1);
    return launch_status("token_logprobs");
}

template <typename T> int forward(const LogprobArgs& a, cudaStream_t st) {
    const bool small = a.vocab <= 512 * Elems<T>::E;
    if (a.top > 0) return small ? launch_forward<T, 128, true>(a, st) : launch_forward<T, 256, true>(a, st);
    return small ? launch_forward<T, 128, false>(a, st) : launch_forward<T, 256, false>(a, st);
}

template <typename T, int THREADS, bool VEC> int launch_backward(const LogprobGradArgs& a, cudaStream_t st) {
    const long long chunks = (a.vocab + Elems<T>::E - 1) / Elems<T>::E + 1;
    const long long segments = (chunks + THREADS * kUnroll - 1) / (THREADS * kUnroll);
    const long long cap = static_cast<long long>(sm_count()) * (1280 / THREADS);
    const long long items = a.rows * segments;
    auto logprobs_grad_kern = token_logprobs_grad_kernel<T, THREADS, VEC>;
    launch_pdl(logprobs_grad_kern, static_cast<unsigned>(items < cap ? items : cap), THREADS, 0, st, a, segments);
    return launch_status("token_logprobs_backward");
}

template <typename T> int backward(const LogprobGradArgs& a, cudaStream_t st) {
    const long long E = Elems<T>::E;
    const auto pl = reinterpret_cast<uintptr_t>(a.logits), pd = reinterpret_cast<uintptr_t>(a.dlogits);
    const bool vec = (pl & 15u) == (pd & 15u) && (a.ld - a.ldd) % E == 0;
    if (!vec) return launch_backward<T, 256, false>(a, st);
    return a.vocab <= 512 * E ? launch_backward<T, 128, true>(a, st) : launch_backward<T, 256, true>(a, st);
}

int check_shape(const char* what, size_t rows, size_t vocab, size_t ld, float temperature, int targets_dt, bool targets) {
    if (vocab == 0 || vocab > 0x40000000u) return fail(cudaErrorInvalidValue, "%s: vocab %zu outside [1, 2^30]", what, vocab);
    if (rows > (size_t{1} << 40)) return fail(cudaErrorInvalidValue, "%s: %zu rows", what, rows);
    if (ld < vocab || ld > (size_t{1} << 40)) return fail(cudaErrorInvalidValue, "%s: row stride %zu below vocab %zu", what, ld, vocab);
    if (!(temperature > 0.f) || !std::isfinite(temperature) || !std::isfinite(kLog2e / temperature))
        return fail(cudaErrorInvalidValue, "%s: temperature must be positive and finite", what);
    if (targets && targets_dt != DT_I32 && targets_dt != DT_I64)
        return fail(cudaErrorInvalidValue, "%s: targets must be I32 or I64", what);
    return 0;
}

bool element_aligned(const void* p, int dt) {
    return (reinterpret_cast<uintptr_t>(p) & (dt == DT_F32 ? 3u : 1u)) == 0;
}

}  // namespace

}  // namespace bee_b200

using namespace bee_b200;

extern "C" {

int bee_b200_token_logprobs(int dt, const void* logits, size_t ld, int targets_dt, const void* targets, size_t rows,
                            size_t vocab, float temperature, float* logprob, float* entropy, float* row_max,
                            float* log_sum, size_t top, int32_t* top_ids, float* top_logprobs, bee_b200_stream_t stream) {
    if (int rc = check_shape("token_logprobs", rows, vocab, ld, temperature, targets_dt, logprob != nullptr)) return rc;
    if (dt != DT_F32 && dt != DT_BF16 && dt != DT_F16) return fail(cudaErrorInvalidValue, "token_logprobs: unsupported dtype %d", dt);
    if (top > kTopMax || top > vocab)
        return fail(cudaErrorInvalidValue, "token_logprobs: %zu alternatives (at most %d and the vocabulary)", top, kTopMax);
    if (rows == 0) return ok();
    if (!logits || (logprob && !targets) || (top > 0 && (!top_ids || !top_logprobs)))
        return fail(cudaErrorInvalidValue, "token_logprobs: null pointer");
    if (!element_aligned(logits, dt)) return fail(cudaErrorInvalidValue, "token_logprobs: logits are not aligned to their type");
    LogprobArgs a{logits, targets, targets_dt == DT_I64 ? 1 : 0, static_cast<long long>(ld), static_cast<long long>(rows),
                  static_cast<long long>(vocab), 1.0f / temperature, static_cast<int>(top), logprob, entropy, row_max, log_sum,
                  top_logprobs, top_ids};
    cudaStream_t st = as_stream(stream);
    if (dt == DT_F32) return forward<float>(a, st);
    if (dt == DT_BF16) return forward<__nv_bfloat16>(a, st);
    return forward<__half>(a, st);
}

int bee_b200_token_logprobs_backward(int dt, const void* logits, size_t ld, int targets_dt, const void* targets, size_t rows,
                                     size_t vocab, float temperature, const float* row_max, const float* log_sum,
                                     const float* entropy, const float* dlogprob, const float* dentropy, void* dlogits,
                                     size_t ldd, bee_b200_stream_t stream) {
    const char* what = "token_logprobs_backward";
    if (int rc = check_shape(what, rows, vocab, ld, temperature, targets_dt, dlogprob != nullptr)) return rc;
    if (dt != DT_F32 && dt != DT_BF16 && dt != DT_F16) return fail(cudaErrorInvalidValue, "%s: unsupported dtype %d", what, dt);
    if (ldd < vocab || ldd > (size_t{1} << 40)) return fail(cudaErrorInvalidValue, "%s: row stride %zu below vocab %zu", what, ldd, vocab);
    if (rows == 0) return ok();
    if (!logits || !dlogits || !row_max || !log_sum || (dlogprob && !targets) || (dentropy && !entropy))
        return fail(cudaErrorInvalidValue, "%s: null pointer", what);
    if (!element_aligned(logits, dt) || !element_aligned(dlogits, dt))
        return fail(cudaErrorInvalidValue, "%s: logits and gradients must be aligned to their type", what);
    if (logits == dlogits && ld != ldd) return fail(cudaErrorInvalidValue, "%s: in place needs equal row strides", what);
    LogprobGradArgs a{logits, targets, targets_dt == DT_I64 ? 1 : 0, static_cast<long long>(ld), static_cast<long long>(ldd),
                      static_cast<long long>(rows), static_cast<long long>(vocab), 1.0f / temperature, row_max, log_sum,
                      entropy, dlogprob, dentropy, dlogits};
    cudaStream_t st = as_stream(stream);
    if (dt == DT_F32) return backward<float>(a, st);
    if (dt == DT_BF16) return backward<__nv_bfloat16>(a, st);
    return backward<__half>(a, st);
}

}  // extern "C"
