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
// Alternatives: a thread's running maximum is also the largest element of its
// share of the row.  The k-th largest of these maxima bounds the row's k-th
// largest element from below, and every element above the bound lies in the
// share of one of the k threads with the largest maxima.  So the stream needs
// no list of candidates: after it, k shares (of a few hundred elements each) are
// read again from L2 and inserted into lists of 32 keys held one per lane.
// Keys are (value, ~index) in 64 bits: ties go to the lowest index.
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
    static __device__ __forceinline__ float max(uint4 q) {
        const float2 m = __bfloat1622float2(__hmax2(__hmax2(h2(q.x), h2(q.y)), __hmax2(h2(q.z), h2(q.w))));
        return fmaxf(m.x, m.y);
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
    static __device__ __forceinline__ float max(uint4 q) {
        const float2 m = __half22float2(__hmax2(__hmax2(h2(q.x), h2(q.y)), __hmax2(h2(q.z), h2(q.w))));
        return fmaxf(m.x, m.y);
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

// One step of a bitonic network over the lanes: the lane keeps the larger key
// of itself and lane ^ d if `up`, else the smaller.
__device__ __forceinline__ uint64_t exchange(uint64_t k, int d, bool up) {
    const uint64_t o = __shfl_xor_sync(0xffffffffu, k, d);
    return ((o > k) == up) ? o : k;
}
// Sorts 32 keys, one per lane, largest first.
__device__ __forceinline__ uint64_t sort_lanes(uint64_t k, int lane) {
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int d = size >> 1; d > 0; d >>= 1) k = exchange(k, d, ((lane & d) == 0) == ((lane & size) == 0));
    return k;
}
// The 32 largest of two lists sorted largest first (keys are distinct, or 0).
__device__ __forceinline__ uint64_t merge_lanes(uint64_t k, const uint64_t* other, int lane) {
    const uint64_t o = other[31 - lane];
    k = o > k ? o : k;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) k = exchange(k, d, (lane & d) == 0);
    return k;
}

// The 32 largest keys of the block's warps' sorted lists, in warp 0 (others: undefined).
template <int WARPS>
__device__ __forceinline__ uint64_t merge_block(uint64_t k, uint64_t (*lists)[32], int warp, int lane) {
#pragma unroll
    for (int half = WARPS / 2; half > 0; half >>= 1) {
        if (warp >= half && warp < 2 * half) lists[warp][lane] = k;
        __syncthreads();
        if (warp < half) k = merge_lanes(k, lists[warp + half], lane);
        __syncthreads();
    }
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
constexpr int kMaxCluster = 8;
constexpr int kStages = 3;  // batches in its part of the shared-memory ring

__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(sm100::smem_u32(dst)), "l"(src) : "memory");
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
    // the thread that reads chunk c
    template <int THREADS> __device__ __forceinline__ int owner(int c) const {
        return c == edge_lo ? 0 : c == edge_hi ? 1 : (c - lo) % THREADS;
    }
};

// Clusters of `cluster` CTAs (1: single CTAs) take rows in grid-stride order.
// Every thread streams its own chunks of the coming batches, across rows, into
// its own slots of a ring with cp.async, so that loads stay in flight while a row
// is joined and its alternatives are sought; no barrier is needed for the ring.
template <typename T, int THREADS, bool TOP>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) token_logprobs_kernel(const LogprobArgs a, int cluster) {
    constexpr int WARPS = THREADS / 32;
    static_assert(2 * WARPS >= kMaxCluster, "a warp of rank 0 joins at most two of the cluster's lists");
    constexpr int E = Elems<T>::E;
    extern __shared__ __align__(16) uint4 ring[];  // [kStages][kUnroll][THREADS]
    __shared__ Stat warp_stat[WARPS];
    __shared__ Stat cta_stat[2][kMaxCluster];                // rank 0's copy is filled by the whole cluster, alternating by row
    __shared__ uint64_t lists[WARPS][32];
    __shared__ uint64_t cta_list[2][TOP ? kMaxCluster : 1][32];
    __shared__ uint64_t owners[32];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = cluster > 1 ? static_cast<int>(sm100::cluster_ctarank()) : 0;
    const float c = a.inv_t * kLog2e;
    if (cluster > 1) sm100::cluster_sync();  // every CTA of the cluster runs before its shared memory is written
    pdl_wait();
    const long long step = gridDim.x / cluster, r0 = blockIdx.x / cluster;

    // the batch to copy next: the issue_at-th chunk of issue_row's part onwards
    long long issue_row = r0;
    int issue_at = tid, issue_hi = 0, issue_slot = 0;
    const uint4* issue_base = nullptr;
    int issue_end = 0;  // uniform: batches left in the row
    auto open_row = [&] {
        if (issue_row >= a.rows) return;
        const Part<T> p(a, issue_row, rank, cluster);
        issue_base = p.row.base;
        issue_at = p.lo + tid;
        issue_hi = p.hi;
        issue_end = (p.hi - p.lo + kUnroll * THREADS - 1) / (kUnroll * THREADS);
    };
    auto issue = [&] {
        while (issue_row < a.rows && issue_end == 0) {  // rows without whole chunks have no batches
            issue_row += step;
            open_row();
        }
        if (issue_row < a.rows) {
#pragma unroll
            for (int j = 0; j < kUnroll; ++j)
                if (issue_at + j * THREADS < issue_hi)
                    cp_async16(ring + (issue_slot * kUnroll + j) * THREADS + tid, issue_base + issue_at + j * THREADS);
            issue_at += kUnroll * THREADS;
            --issue_end;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");  // empty past the end: the wait counts stay uniform
        issue_slot = issue_slot + 1 == kStages ? 0 : issue_slot + 1;
    };
    open_row();
    for (int j = 1; j < kStages; ++j) issue();

    int slot = 0, turn = 0;
    for (long long r = r0; r < a.rows; r += step, turn ^= 1) {
        if (r + step >= a.rows) pdl_trigger();  // this CTA's last row
        const Part<T> part(a, r, rank, cluster);
        const RowChunks<T>& row = part.row;

        // early loads: the target's logit (by the thread that writes the row's results) and the partial chunks
        long long target = -1;
        float xt = -INFINITY;
        if (tid == 0 && rank == 0 && a.logprob) {
            target = target_of(a.targets, a.targets_i64, r);
            xt = target < 0 ? 0.f : target < a.vocab ? Elems<T>::get(row.row + target) : NAN;
        }
        const int edge = tid == 0 ? part.edge_lo : tid == 1 ? part.edge_hi : -1;
        uint4 edge_chunk = Elems<T>::fill();
        if (edge >= 0) edge_chunk = row.partial(edge);

        Stat st{-INFINITY, 0.f, 0.f};
        int at = -1;  // the chunk that holds this thread's maximum
        auto consume = [&](const uint4 (&q)[kUnroll], int c0, int count) {
            float cm[kUnroll], bm = -INFINITY;
#pragma unroll
            for (int j = 0; j < kUnroll; ++j) {
                cm[j] = Elems<T>::max(q[j]);
                bm = fmaxf(bm, cm[j]);
            }
            // the partial first chunk comes last but holds the lowest indices: it wins a tie
            if (bm > st.m || at < 0 || (TOP && c0 == part.edge_lo && bm == st.m)) {
                rebase(st, bm, c);
                at = c0;
                if (TOP) {
#pragma unroll
                    for (int j = kUnroll - 1; j >= 0; --j)
                        if (j < count && cm[j] == bm) at = c0 + j * THREADS;
                }
            }
            const float m = finite_max(st.m);
            const uint64_t negm2 = pack_f32x2(-m, -m), c2 = pack_f32x2(c, c);
            uint64_t s2 = 0, z2 = 0;  // pairs of fp32 zeros
#pragma unroll
            for (int j = 0; j < kUnroll; ++j) {
                float v[E];
                Elems<T>::unpack(q[j], v);
#pragma unroll
                for (int e = 0; e < E; e += 2) {
                    float lo, hi;
                    unpack_f32x2(mul_f32x2(add_f32x2(pack_f32x2(v[e], v[e + 1]), negm2), c2), lo, hi);
                    lo = max_nan(lo, kZFloor);
                    hi = max_nan(hi, kZFloor);
                    const uint64_t e2 = pack_f32x2(ex2(lo), ex2(hi));
                    s2 = add_f32x2(s2, e2);
                    z2 = fma_f32x2(e2, pack_f32x2(lo, hi), z2);
                }
            }
            float lo, hi;
            unpack_f32x2(s2, lo, hi);
            st.s += lo + hi;
            unpack_f32x2(z2, lo, hi);
            st.z += lo + hi;
        };
        for (int c0 = part.lo; c0 < part.hi; c0 += kUnroll * THREADS) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
            issue();
            const uint4* mine = ring + slot * kUnroll * THREADS + tid;
            slot = slot + 1 == kStages ? 0 : slot + 1;
            const int left = part.hi - c0 - tid;  // this thread's chunks are those at 0, THREADS, ... below `left`
            if (left <= 0) continue;
            uint4 q[kUnroll];
            if (left > (kUnroll - 1) * THREADS) {
#pragma unroll
                for (int j = 0; j < kUnroll; ++j) q[j] = mine[j * THREADS];
                consume(q, c0 + tid, kUnroll);
            } else {
#pragma unroll
                for (int j = 0; j < kUnroll; ++j) q[j] = j * THREADS < left ? mine[j * THREADS] : Elems<T>::fill();
                consume(q, c0 + tid, (left + THREADS - 1) / THREADS);
            }
        }
        if (edge >= 0) {
            uint4 q[kUnroll];
            q[0] = edge_chunk;
#pragma unroll
            for (int j = 1; j < kUnroll; ++j) q[j] = Elems<T>::fill();
            consume(q, edge, 1);
        }
        __syncwarp();

        uint64_t best = 0;
        if constexpr (TOP) {
            // owners of the k largest thread maxima
            uint64_t key = at >= 0 ? make_key(st.m, static_cast<uint32_t>(at)) : 0;
            key = merge_block<WARPS>(sort_lanes(key, lane), lists, warp, lane);
            if (warp == 0) owners[lane] = key;
            __syncthreads();
            const uint32_t bound = static_cast<uint32_t>(owners[a.top - 1] >> 32);  // 0 if fewer threads hold anything
            // inserts the elements of each lane's chunk (index cc; none where !in) into the warp's sorted list
            auto insert = [&](uint4 chunk, int cc, bool in) {
                float v[E];
                Elems<T>::unpack(chunk, v);
                const long long i0 = row.first(cc);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const bool real = in && i0 + e >= 0 && i0 + e < row.n && v[e] == v[e] && ordered(v[e]) >= bound;
                    if (!__any_sync(0xffffffffu, real)) continue;
                    const uint64_t ck = real ? make_key(v[e], static_cast<uint32_t>(i0 + e)) : 0;
                    uint32_t todo = __ballot_sync(0xffffffffu, ck > __shfl_sync(0xffffffffu, best, 31));
                    while (todo) {
                        const int src = __ffs(todo) - 1;
                        todo &= todo - 1;
                        const uint64_t nk = __shfl_sync(0xffffffffu, ck, src);
                        const int pos = __popc(__ballot_sync(0xffffffffu, best > nk));
                        const uint64_t up = __shfl_up_sync(0xffffffffu, best, 1);
                        best = lane < pos ? best : lane == pos ? nk : up;
                    }
                }
            };
            for (int j = warp; j < a.top; j += WARPS) {
                const uint64_t o = owners[j];
                if (o == 0) break;  // the list is sorted: no more owners
                const int owner = part.template owner<THREADS>(static_cast<int>(~static_cast<uint32_t>(o)));
                for (int cb = part.lo + owner; cb < part.hi; cb += 32 * THREADS) {
                    const int cc = cb + lane * THREADS;
                    insert(cc < part.hi ? __ldg(row.base + cc) : Elems<T>::fill(), cc, cc < part.hi);
                }
                const int partial = owner == 0 ? part.edge_lo : owner == 1 ? part.edge_hi : -1;
                if (partial >= 0) insert(lane == 0 ? row.partial(partial) : Elems<T>::fill(), partial, lane == 0);
            }
        }

        // join the block's statistics, then the cluster's, each in a fixed order
        st = warp_join(st, c);
        if (lane == 0) warp_stat[warp] = st;
        if constexpr (TOP) best = merge_block<WARPS>(best, lists, warp, lane);
        __syncthreads();
        if (warp == 0) st = warp_join(lane < WARPS ? warp_stat[lane] : Stat{-INFINITY, 0.f, 0.f}, c);
        if (cluster > 1) {
            if (warp == 0) {
                const uint32_t dst = sm100::mapa_shared(sm100::smem_u32(&cta_stat[turn][rank]), 0);
                if (lane < 3) {
                    const float v = lane == 0 ? st.m : lane == 1 ? st.s : st.z;
                    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst + 4 * lane), "f"(v) : "memory");
                }
                if constexpr (TOP) {
                    const uint32_t dk = sm100::mapa_shared(sm100::smem_u32(&cta_list[turn][rank][lane]), 0);
                    asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(dk), "l"(best) : "memory");
                }
            }
            __syncwarp();
            sm100::cluster_sync();  // the other of the two buffers has been read: rank 0 came past its reads to get here
            if (rank == 0) {
                if (warp == 0) st = warp_join(lane < cluster ? cta_stat[turn][lane] : Stat{-INFINITY, 0.f, 0.f}, c);
                if constexpr (TOP) {
                    best = warp < cluster ? cta_list[turn][warp][lane] : 0;
                    if (WARPS < kMaxCluster && warp + WARPS < cluster) best = merge_lanes(best, cta_list[turn][warp + WARPS], lane);
                    best = merge_block<WARPS>(best, lists, warp, lane);
                }
            }
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
    const float gl = g.target >= 0 ? a.dlogprob[r] : 0.f;
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
int cluster_for(long long rows, long long chunks, long long slots) {
    int best = 1;
    double least = 0, joins = 1024;
    for (int cl = 1; cl <= kMaxCluster; cl *= 2, joins += 128) {
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
    const int cl = cluster_for(a.rows, chunks, slots);
    const size_t smem = sizeof(uint4) * kStages * kUnroll * THREADS;
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
