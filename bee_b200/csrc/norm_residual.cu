// The step from one block's output to the next block's input, in one pass, and
// its gradient:
//   n  = h rstd(h) w_post            (n = h without w_post)
//   x' = alpha x + beta gate n       (gate: one row, or one row per group of rows)
//   y  = x' rstd(x') w_pre
// with rstd(v) = 1 / sqrt(mean(v^2) + eps) over a row.  New: the reference has
// no normalisation; rms_norm_rows is the unfused form.
//
// Backward, from the forward's inputs and the gradients dx', dy of its outputs
// (statistics and x' are recomputed, nothing has to be kept):
//   xh = x' rstd(x'),  D = dx' + rstd(x') (dy w_pre - xh mean(dy w_pre xh))
//   dx = alpha D,      dn = beta gate D,      hh = h rstd(h)
//   dh = rstd(h) (dn w_post - hh mean(dn w_post hh))
//   dw_pre = sum_rows dy xh,  dw_post = sum_rows dn hh,  dgate = sum_group beta D n
//
// Both are bound by HBM (forward: 2 reads and 2 writes of the tensor, backward:
// 4 and 2).  A CTA owns whole rows, so every tensor crosses HBM once: upcoming
// rows are copied into a shared-memory ring with cp.async while the current one
// is reduced; the sum of squares of the next row's h joins a sum of the current
// row, so that a row costs one block reduction forward and two backward.  All arithmetic is
// fp32, in packed pairs; results are rounded once, when stored.
//
// A thread owns the same kEpt = 16 columns of every row, so the backward's column
// sums stay in registers over the CTA's contiguous range of rows; each CTA
// writes one row of partial sums and a second kernel adds them in a fixed order
// (results do not depend on timing).  A group of rows that lies inside one
// CTA's range is finished there; one that is cut leaves a partial per CTA.
//
// Rows of any length up to 16384 (fp32: 12288): if it is a whole number of 16-byte vectors and
// all tensors are 16-byte aligned, each thread copies and reads only its own
// vectors (no barrier for the ring); otherwise the block copies the aligned
// 16-byte blocks that cover the row and threads read single elements from them.
#include <cmath>
#include <type_traits>

#include "common.cuh"
#include "sm100.cuh"

namespace bee_b200 {

namespace {

constexpr int kEpt = 16;         // columns per thread
constexpr int kPairs = kEpt / 2;
// 1024 threads' columns; in fp32 768 threads', since the four rows of a backward slot fill the shared memory
constexpr size_t max_cols(int dt) { return dt == DT_F32 ? 12288 : 16384; }
using f2 = uint64_t;             // two fp32 values

__device__ __forceinline__ f2 dup(float v) { return pack_f32x2(v, v); }
__device__ __forceinline__ float hsum(f2 v) {
    float a, b;
    unpack_f32x2(v, a, b);
    return a + b;
}

template <typename T> struct Conv;
template <> struct Conv<float> {
    static __device__ __forceinline__ float up(float v) { return v; }
    static __device__ __forceinline__ float down(float v) { return v; }
};
template <> struct Conv<__nv_bfloat16> {
    static __device__ __forceinline__ float up(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 down(float v) { return __float2bfloat16_rn(v); }
    static __device__ __forceinline__ f2 up2(uint32_t w) { return bf16x2_to_f32x2(w); }
    static __device__ __forceinline__ uint32_t down2(f2 v) { return f32x2_to_bf16x2(v); }
};
template <> struct Conv<__half> {
    static __device__ __forceinline__ float up(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half down(float v) { return __float2half_rn(v); }
    static __device__ __forceinline__ f2 up2(uint32_t w) {
        const float2 f = __half22float2(*reinterpret_cast<__half2*>(&w));
        return pack_f32x2(f.x, f.y);
    }
    static __device__ __forceinline__ uint32_t down2(f2 v) {
        float a, b;
        unpack_f32x2(v, a, b);
        return pack_f16x2(a, b);
    }
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Waits until at most `pending` (0 or 1: a ring has up to three slots) of the thread's groups are in flight.
__device__ __forceinline__ void cp_wait(int pending) {
    if (pending == 0) asm volatile("cp.async.wait_group 0;" ::: "memory");
    else asm volatile("cp.async.wait_group 1;" ::: "memory");
}

// The columns of one thread.  VEC: 16-byte vectors tid, tid + THREADS, ...;
// otherwise columns tid, tid + THREADS, ....  Columns past the row read as 0
// and are not written, so they add nothing to any sum.
template <typename T, bool VEC, int THREADS> struct Cols {
    [[maybe_unused]] static constexpr int E = 16 / sizeof(T);
    uint32_t cols;
    __device__ __forceinline__ explicit Cols(uint32_t n) : cols(n) {}
    __device__ __forceinline__ static uint32_t vec(int j) { return j * THREADS + threadIdx.x; }
    __device__ __forceinline__ static uint32_t col(int k) { return k * THREADS + threadIdx.x; }

    static __device__ __forceinline__ void unpack(uint4 q, f2* v) {
        if constexpr (std::is_same_v<T, float>) {
            v[0] = pack_f32x2(__uint_as_float(q.x), __uint_as_float(q.y));
            v[1] = pack_f32x2(__uint_as_float(q.z), __uint_as_float(q.w));
        } else {
            v[0] = Conv<T>::up2(q.x); v[1] = Conv<T>::up2(q.y); v[2] = Conv<T>::up2(q.z); v[3] = Conv<T>::up2(q.w);
        }
    }
    static __device__ __forceinline__ uint4 pack(const f2* v) {
        if constexpr (std::is_same_v<T, float>) {
            float a, b, c, d;
            unpack_f32x2(v[0], a, b);
            unpack_f32x2(v[1], c, d);
            return make_uint4(__float_as_uint(a), __float_as_uint(b), __float_as_uint(c), __float_as_uint(d));
        } else {
            return make_uint4(Conv<T>::down2(v[0]), Conv<T>::down2(v[1]), Conv<T>::down2(v[2]), Conv<T>::down2(v[3]));
        }
    }
    // Slots as wide as the block's columns, zero past the row's end, so that they are read without bounds; the
    // widest rows have exact ones.  Bytes of a row in a slot (its first 16-byte block may begin before the row):
    static constexpr bool kPadded = THREADS < 1024;
    static __host__ __device__ constexpr uint32_t pitch(uint32_t cols) {
        return (kPadded ? THREADS * kEpt * static_cast<uint32_t>(sizeof(T)) : (cols * static_cast<uint32_t>(sizeof(T)) + 15) / 16 * 16) + (VEC ? 0 : 16);
    }
    // zeros in a slot: VEC, this thread's own vectors past the row's end; else this thread's share of all of it
    __device__ __forceinline__ void pad(uint8_t* slot) const {
        if constexpr (kPadded && VEC) {
#pragma unroll
            for (int j = 0; j < kEpt / E; ++j)
                if (vec(j) * E >= cols) reinterpret_cast<uint4*>(slot)[vec(j)] = make_uint4(0, 0, 0, 0);
        } else if constexpr (kPadded) {
            for (uint32_t i = threadIdx.x; i < pitch(cols) / 16; i += THREADS) reinterpret_cast<uint4*>(slot)[i] = make_uint4(0, 0, 0, 0);
        }
    }
    // this thread's columns of an optional vector into a slot (absent: ones), which only this thread reads
    __device__ __forceinline__ void keep(T* slot, const T* w) const {
        f2 v[kPairs];
        if (w) {
            read<true>(w, v);
        } else {
#pragma unroll
            for (int k = 0; k < kPairs; ++k) v[k] = dup(1.f);
        }
        if constexpr (VEC) {
#pragma unroll
            for (int j = 0; j < kEpt / E; ++j)
                if (kPadded || vec(j) * E < cols) reinterpret_cast<uint4*>(slot)[vec(j)] = pack(v + j * (E / 2));
        } else {
#pragma unroll
            for (int k = 0; k < kPairs; ++k) {
                float a, b;
                unpack_f32x2(v[k], a, b);
                if (kPadded || col(2 * k) < cols) slot[col(2 * k)] = Conv<T>::down(a);
                if (kPadded || col(2 * k + 1) < cols) slot[col(2 * k + 1)] = Conv<T>::down(b);
            }
        }
    }
    // from a row (shared or global memory; LDG: read-only global vectors)
    template <bool LDG> __device__ __forceinline__ void read(const T* p, f2 (&v)[kPairs]) const {
        if constexpr (kPadded && VEC && !LDG) {
#pragma unroll
            for (int j = 0; j < kEpt / E; ++j) unpack(reinterpret_cast<const uint4*>(p)[vec(j)], v + j * (E / 2));
        } else if constexpr (kPadded && !LDG) {
#pragma unroll
            for (int k = 0; k < kPairs; ++k) v[k] = pack_f32x2(Conv<T>::up(p[col(2 * k)]), Conv<T>::up(p[col(2 * k + 1)]));
        } else if constexpr (VEC) {
#pragma unroll
            for (int j = 0; j < kEpt / E; ++j) {
                const uint4* q = reinterpret_cast<const uint4*>(p) + vec(j);
                unpack(vec(j) * E < cols ? (LDG ? __ldg(q) : *q) : make_uint4(0, 0, 0, 0), v + j * (E / 2));
            }
        } else {
#pragma unroll
            for (int k = 0; k < kPairs; ++k)
                v[k] = pack_f32x2(col(2 * k) < cols ? Conv<T>::up(p[col(2 * k)]) : 0.f,
                                  col(2 * k + 1) < cols ? Conv<T>::up(p[col(2 * k + 1)]) : 0.f);
        }
    }
    // an optional vector of weights; absent: ones
    __device__ __forceinline__ void weights(const T* p, f2 (&v)[kPairs]) const {
        if (p) {
            read<true>(p, v);
        } else {
#pragma unroll
            for (int k = 0; k < kPairs; ++k) v[k] = dup(1.f);
        }
    }
    __device__ __forceinline__ void write(T* p, const f2 (&v)[kPairs]) const {
        if constexpr (VEC) {
#pragma unroll
            for (int j = 0; j < kEpt / E; ++j)
                if (vec(j) * E < cols) __stcs(reinterpret_cast<uint4*>(p) + vec(j), pack(v + j * (E / 2)));
        } else {
#pragma unroll
            for (int k = 0; k < kPairs; ++k) {
                float a, b;
                unpack_f32x2(v[k], a, b);
                if (col(2 * k) < cols) p[col(2 * k)] = Conv<T>::down(a);
                if (col(2 * k + 1) < cols) p[col(2 * k + 1)] = Conv<T>::down(b);
            }
        }
    }
    // fp32 partial sums (p 16-byte aligned)
    __device__ __forceinline__ void write_f32(float* p, const f2 (&v)[kPairs]) const {
        if constexpr (VEC) {
#pragma unroll
            for (int k = 0; k < kPairs; k += 2) {
                const uint32_t c = vec(2 * k / E) * E + 2 * k % E;
                float4 q;
                unpack_f32x2(v[k], q.x, q.y);
                unpack_f32x2(v[k + 1], q.z, q.w);
                if (c < cols) *reinterpret_cast<float4*>(p + c) = q;
            }
        } else {
#pragma unroll
            for (int k = 0; k < kPairs; ++k) {
                float a, b;
                unpack_f32x2(v[k], a, b);
                if (col(2 * k) < cols) p[col(2 * k)] = a;
                if (col(2 * k + 1) < cols) p[col(2 * k + 1)] = b;
            }
        }
    }
    __device__ __forceinline__ void read_f32(const float* p, f2 (&v)[kPairs]) const {
#pragma unroll
        for (int k = 0; k < kPairs; ++k) {
            const uint32_t ca = VEC ? vec(2 * k / E) * E + 2 * k % E : col(2 * k);
            const uint32_t cb = VEC ? ca + 1 : col(2 * k + 1);
            v[k] = pack_f32x2(ca < cols ? p[ca] : 0.f, cb < cols ? p[cb] : 0.f);
        }
    }
};

// Two sums over the block with one barrier: consecutive calls use alternating rows
// of `red`, so a call's writes never meet the previous call's reads.
template <int THREADS> struct BlockSum {
    static constexpr int WARPS = (THREADS / 32 + 3) / 4 * 4;  // those past the block's add 0
    f2 (*red)[WARPS];  // two rows of the warps' two sums
    int parity = 0;
    __device__ __forceinline__ explicit BlockSum(f2 (*r)[WARPS]) : red(r) {
        if constexpr (THREADS / 32 < WARPS) {
            for (int i = threadIdx.x; i < 2 * WARPS; i += THREADS) r[i / WARPS][i % WARPS] = 0;
            __syncthreads();
        }
    }
    // of a and b, at once
    __device__ __forceinline__ float2 operator()(float a, float b) {
        a = warp_sum(a);
        b = warp_sum(b);
        if constexpr (THREADS == 32) return make_float2(a, b);
        if ((threadIdx.x & 31) == 0) red[parity][threadIdx.x >> 5] = pack_f32x2(a, b);
        __syncthreads();
        f2 r = 0;
#pragma unroll
        for (int w = 0; w < WARPS; w += 2) {
            const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(&red[parity][w]);
            r = add_f32x2(add_f32x2(r, v.x), v.y);
        }
        parity ^= 1;
        float2 s;
        unpack_f32x2(r, s.x, s.y);
        return s;
    }
};

// A ring of `stages` slots, each one row of up to NT tensors.
template <typename T, bool VEC, int THREADS, int NT> struct Ring {
    const T* src[NT];
    uint8_t* base;
    uint32_t cols, pitch, stages;  // pitch: bytes of one tensor's row in a slot
    long long row, end;            // next row to copy
    uint32_t slot = 0;             // its slot

    __device__ __forceinline__ uint8_t* at(uint32_t s, int t) const { return base + (s * NT + t) * pitch; }
    // bytes of tensor t's row r that precede it in its slot
    __device__ __forceinline__ uint32_t lead(int t, long long r) const {
        return VEC ? 0u : static_cast<uint32_t>(reinterpret_cast<uintptr_t>(src[t] + r * cols) & 15u);
    }
    __device__ __forceinline__ const T* read(uint32_t s, int t, long long r) const {
        return reinterpret_cast<const T*>(at(s, t) + lead(t, r));
    }
    __device__ __forceinline__ void issue() {
        if (row < end) {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                if (!src[t]) continue;
                const T* g = src[t] + row * cols;
                if constexpr (VEC) {
                    constexpr uint32_t E = 16 / sizeof(T);
                    const uint32_t dst = sm100::smem_u32(at(slot, t));
#pragma unroll
                    for (int j = 0; j < kEpt / static_cast<int>(E); ++j) {
                        const uint32_t v = j * THREADS + threadIdx.x;
                        if (v * E < cols) cp_async16(dst + v * 16, reinterpret_cast<const uint4*>(g) + v, 16);
                    }
                } else {
                    // the 16-byte blocks that cover the row; the last is cut at the row's end (zeros follow), one
                    // that begins before the tensor is copied element by element, and one of zeros comes after
                    // them: the row before may have ended later in this slot, by less than a block
                    const uint32_t ld = lead(t, row), bytes = ld + cols * static_cast<uint32_t>(sizeof(T));
                    const uint8_t* a = reinterpret_cast<const uint8_t*>(g) - ld;
                    const uint32_t filled = (bytes + 15) / 16 * 16 + 16;
                    for (uint32_t o = threadIdx.x * 16; o < (filled < pitch ? filled : pitch); o += THREADS * 16) {
                        if (o == 0 && row == 0 && ld != 0) {
                            for (uint32_t b = ld; b < 16 && b < bytes; b += sizeof(T))
                                *reinterpret_cast<T*>(at(slot, t) + b) = *reinterpret_cast<const T*>(a + b);
                        } else {
                            // (a block of zeros reads nothing; its address is the row's)
                            const uint32_t n = o >= bytes ? 0 : bytes - o < 16 ? bytes - o : 16;
                            cp_async16(sm100::smem_u32(at(slot, t) + o), n ? a + o : a, n);
                        }
                    }
                }
            }
        }
        cp_commit();  // one group per row, empty past the end, so that the wait counts stay uniform
        ++row;
        slot = slot + 1 == stages ? 0 : slot + 1;
    }
    // Waits for the current row's copies and starts those of a later row in the slot that is free by then.
    __device__ __forceinline__ void advance() {
        if (stages == 1) {
            if constexpr (!VEC) __syncthreads();
            issue();
            cp_wait(0);
            if constexpr (!VEC) __syncthreads();
        } else {
            cp_wait(static_cast<int>(stages) - 2);
            if constexpr (!VEC) __syncthreads();  // the row is complete, and its predecessor's slot has been read by all
            issue();
        }
    }
    template <typename C> __device__ __forceinline__ void start(const C& cl) {
        for (uint32_t s = 0; s < stages; ++s)
            for (int t = 0; t < NT; ++t) cl.pad(at(s, t));
        if constexpr (!VEC) __syncthreads();
        for (uint32_t s = 1; s < stages; ++s) issue();
    }
};

struct NormArgs {
    const void *h, *x, *w_post, *gate, *w_pre;
    void *x_out, *y;
    const void *dx_out, *dy;
    void *dh, *dx, *dgate;
    float *part_post, *part_pre, *part_gate;  // partial sums: [ctas][part], [ctas][part], [2 * ctas][part]
    long long rows, per_cta, group;           // group: rows per gate row
    uint32_t cols, part, pitch, stages;       // part: cols rounded up to 4
    float alpha, beta, eps;
};

// ---------------------------------------------------------------- forward

// The vectors come from L1 for every row: holding beta gate w_post and w_pre in
// registers leaves three quarters of the threads (32768 x 4096 bf16, cold caches: 191 us, 186 so).
template <typename T, bool VEC, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) norm_residual_kernel(const NormArgs a) {
    extern __shared__ __align__(16) uint8_t ring_smem[];
    __shared__ __align__(16) f2 red[2][BlockSum<THREADS>::WARPS];
    BlockSum<THREADS> block_sum(red);
    const Cols<T, VEC, THREADS> cl(a.cols);
    const long long r0 = blockIdx.x * a.per_cta;
    const long long r1 = r0 + a.per_cta < a.rows ? r0 + a.per_cta : a.rows;
    const T *wpost = static_cast<const T*>(a.w_post), *wpre = static_cast<const T*>(a.w_pre), *gate = static_cast<const T*>(a.gate);
    const float inv_n = 1.0f / static_cast<float>(a.cols);
    Ring<T, VEC, THREADS, 2> ring{{static_cast<const T*>(a.h), static_cast<const T*>(a.x)}, ring_smem, a.cols, a.pitch, a.stages, r0, r1};
    long long group = r0 / a.group, group_end = (group + 1) * a.group;
    // beta gate w_post of the current group
    auto load_factor = [&](f2 (&f)[kPairs]) {
        f2 t[kPairs];
        cl.weights(wpost, f);
        cl.weights(gate ? gate + group * a.cols : nullptr, t);
#pragma unroll
        for (int k = 0; k < kPairs; ++k) f[k] = mul_f32x2(f[k], mul_f32x2(t[k], dup(a.beta)));
    };
    auto squares = [&](const T* row) {
        f2 v[kPairs], ss = 0;
        cl.template read<false>(row, v);
#pragma unroll
        for (int k = 0; k < kPairs; ++k) ss = fma_f32x2(v[k], v[k], ss);
        return hsum(ss);
    };
    pdl_wait();
    ring.start(cl);
    uint32_t slot = 0;
    float rh = 1.f;  // rstd(h) of the current row; found with the sums of the row before
    ring.advance();
    // (as the second of two sums, like every other row's: a row's results do not depend on the rows around it)
    if (wpost) rh = rsqrtf(fmaf(block_sum(0.f, squares(ring.read(0, 0, r0))).y, inv_n, a.eps));
    for (long long r = r0; r < r1; ++r) {
        const bool more = r + 1 < r1;
        if (!more) pdl_trigger();
        f2 v[kPairs], t[kPairs], w[kPairs];
        load_factor(w);
        cl.template read<false>(ring.read(slot, 0, r), v);
        cl.template read<false>(ring.read(slot, 1, r), t);
        f2 ss = 0;
#pragma unroll
        for (int k = 0; k < kPairs; ++k) {
            v[k] = fma_f32x2(mul_f32x2(v[k], dup(rh)), w[k], mul_f32x2(t[k], dup(a.alpha)));
            ss = fma_f32x2(v[k], v[k], ss);
        }
        cl.write(static_cast<T*>(a.x_out) + r * a.cols, v);
        // on to the next row (this one's slot has been read), whose sum of squares joins this row's
        slot = slot + 1 == a.stages ? 0 : slot + 1;
        if (more) ring.advance();
        if (wpre || wpost) {
            const float2 sum = block_sum(hsum(ss), more && wpost ? squares(ring.read(slot, 0, r + 1)) : 0.f);
            if (wpost) rh = rsqrtf(fmaf(sum.y, inv_n, a.eps));
            if (wpre) {
                const f2 rx = dup(rsqrtf(fmaf(sum.x, inv_n, a.eps)));
                cl.weights(wpre, w);
#pragma unroll
                for (int k = 0; k < kPairs; ++k) v[k] = mul_f32x2(mul_f32x2(v[k], rx), w[k]);
                cl.write(static_cast<T*>(a.y) + r * a.cols, v);
            }
        }
        if (r + 1 == group_end) {
            ++group;
            group_end += a.group;
        }
    }
    cp_wait(0);
}

// ---------------------------------------------------------------- backward

// Whether the backward keeps beta gate w_post (in fp32) and w_pre in shared memory:
// L1 misses the vectors beside the rings, and each use would unpack and multiply them
// again (8192 x 4096 fp32: 144 us without, 135 with).  The widest rows need the room for the ring.
template <typename T> constexpr bool keep_vectors(int threads) { return threads < (sizeof(T) == 2 ? 1024 : 768); }

// w_post and the gate share a column sum: with P = sum over a group's rows of D hh,
// dgate = beta w_post P, and dw_post is the sum over the groups of beta gate P.
// From 768 threads on the column sums leave too few registers and some spill
// (4096 x 12288 bf16: 201 us with 768 threads, 295 with 1024, 549 with the sums in memory).
template <typename T, bool VEC, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS <= 512 ? 512 / THREADS : 1) norm_residual_grad_kernel(const NormArgs a) {
    constexpr bool KEEP = keep_vectors<T>(THREADS);
    extern __shared__ __align__(16) uint8_t ring_smem[];
    __shared__ __align__(16) f2 red[2][BlockSum<THREADS>::WARPS];
    BlockSum<THREADS> block_sum(red);
    const Cols<T, VEC, THREADS> cl(a.cols);
    const long long r0 = blockIdx.x * a.per_cta;
    const long long r1 = r0 + a.per_cta < a.rows ? r0 + a.per_cta : a.rows;
    const T *wpost = static_cast<const T*>(a.w_post), *wpre = static_cast<const T*>(a.w_pre);
    const T* gate = static_cast<const T*>(a.gate);
    const float inv_n = 1.0f / static_cast<float>(a.cols);
    Ring<T, VEC, THREADS, 4> ring{{static_cast<const T*>(a.h), static_cast<const T*>(a.x), static_cast<const T*>(a.dx_out),
                                   static_cast<const T*>(a.dy)}, ring_smem, a.cols, a.pitch, a.stages, r0, r1};
    float* my_post = a.part_post + static_cast<long long>(blockIdx.x) * a.part;
    float* my_pre = a.part_pre + static_cast<long long>(blockIdx.x) * a.part;
    float* my_gate = a.part_gate + static_cast<long long>(blockIdx.x) * 2 * a.part;
    f2 s_col[kPairs], s_pre[kPairs];  // sums of D hh (this group's rows) and of dy xh
#pragma unroll
    for (int k = 0; k < kPairs; ++k) s_col[k] = s_pre[k] = 0;
    // KEEP: after the ring, w_pre and then beta gate w_post, of which a thread reads only what it wrote
    T* kept_pre = reinterpret_cast<T*>(ring_smem + a.pitch * 4 * a.stages);
    ulonglong2* kept_factor = reinterpret_cast<ulonglong2*>(ring_smem + a.pitch * (4 * a.stages + 1)) + threadIdx.x;
    long long group = gate ? r0 / a.group : 0;
    long long group_end = gate ? (group + 1) * a.group : r1;
    // beta gate w_post of the current group, from global memory
    auto load_factor = [&](f2 (&f)[kPairs]) {
        f2 t[kPairs];
        cl.weights(wpost, f);
        cl.weights(gate ? gate + group * a.cols : nullptr, t);
#pragma unroll
        for (int k = 0; k < kPairs; ++k) f[k] = mul_f32x2(f[k], mul_f32x2(t[k], dup(a.beta)));
    };
    auto keep_factor = [&] {
        f2 f[kPairs];
        load_factor(f);
#pragma unroll
        for (int k = 0; k < kPairs; k += 2) kept_factor[k / 2 * THREADS] = make_ulonglong2(f[k], f[k + 1]);
    };
    auto factor = [&](f2 (&f)[kPairs]) {
        if constexpr (KEEP) {
#pragma unroll
            for (int k = 0; k < kPairs; k += 2) {
                const ulonglong2 q = kept_factor[k / 2 * THREADS];
                f[k] = q.x;
                f[k + 1] = q.y;
            }
        } else {
            load_factor(f);
        }
    };
    auto squares = [&](const T* row) {
        f2 v[kPairs], ss = 0;
        cl.template read<false>(row, v);
#pragma unroll
        for (int k = 0; k < kPairs; ++k) ss = fma_f32x2(v[k], v[k], ss);
        return hsum(ss);
    };
    pdl_wait();
    ring.start(cl);
    if constexpr (KEEP) {
        cl.keep(kept_pre, wpre);
        keep_factor();
    }
    bool first_group = true;
    uint32_t slot = 0;
    float rh = 1.f;  // of the current row; found with the sums of the row before
    ring.advance();
    // (as the second of two sums, like every other row's: a row's results do not depend on the rows around it)
    if (wpost) rh = rsqrtf(fmaf(block_sum(0.f, squares(ring.read(0, 0, r0))).y, inv_n, a.eps));
    for (long long r = r0; r < r1; ++r) {
        f2 hh[kPairs], v[kPairs], w[kPairs], t[kPairs];
        // hh = h rstd(h), v = x'
        cl.template read<false>(ring.read(slot, 0, r), hh);
        factor(w);
        cl.template read<false>(ring.read(slot, 1, r), t);
#pragma unroll
        for (int k = 0; k < kPairs; ++k) {
            hh[k] = mul_f32x2(hh[k], dup(rh));
            v[k] = fma_f32x2(hh[k], w[k], mul_f32x2(t[k], dup(a.alpha)));
        }
        // v = D
        if (wpre) {
            cl.template read<false>(ring.read(slot, 3, r), t);
            if constexpr (KEEP) cl.template read<false>(kept_pre, w);
            else cl.weights(wpre, w);
            f2 ss = 0, dot = 0;
#pragma unroll
            for (int k = 0; k < kPairs; ++k) {
                ss = fma_f32x2(v[k], v[k], ss);
                w[k] = mul_f32x2(t[k], w[k]);
                dot = fma_f32x2(w[k], v[k], dot);
            }
            const float2 sum = block_sum(hsum(ss), hsum(dot));
            const float rx = rsqrtf(fmaf(sum.x, inv_n, a.eps));
            const f2 rx2 = dup(rx), mean = dup(-rx * sum.y * inv_n);  // -mean(dy w_pre xh)
#pragma unroll
            for (int k = 0; k < kPairs; ++k) {
                const f2 xh = mul_f32x2(v[k], rx2);
                s_pre[k] = fma_f32x2(t[k], xh, s_pre[k]);
                v[k] = mul_f32x2(fma_f32x2(xh, mean, w[k]), rx2);
            }
        } else {
#pragma unroll
            for (int k = 0; k < kPairs; ++k) v[k] = 0;
        }
        if (a.dx_out) {
            cl.template read<false>(ring.read(slot, 2, r), t);
#pragma unroll
            for (int k = 0; k < kPairs; ++k) v[k] = add_f32x2(v[k], t[k]);
        }
#pragma unroll
        for (int k = 0; k < kPairs; ++k) t[k] = mul_f32x2(v[k], dup(a.alpha));
        cl.write(static_cast<T*>(a.dx) + r * a.cols, t);
        // the group's column sum, and v = dn w_post with dn = beta gate D
        factor(w);
        f2 dot = 0;
#pragma unroll
        for (int k = 0; k < kPairs; ++k) {
            s_col[k] = fma_f32x2(v[k], hh[k], s_col[k]);
            v[k] = mul_f32x2(v[k], w[k]);
            dot = fma_f32x2(v[k], hh[k], dot);
        }
        // on to the next row (this one's slot has been read), whose sum of squares joins this row's last sum
        const bool more = r + 1 < r1;
        slot = slot + 1 == a.stages ? 0 : slot + 1;
        if (more) ring.advance();
        if (wpost) {
            const float2 sum = block_sum(hsum(dot), more ? squares(ring.read(slot, 0, r + 1)) : 0.f);
            const f2 mean = dup(-sum.x * inv_n);
#pragma unroll
            for (int k = 0; k < kPairs; ++k) v[k] = mul_f32x2(fma_f32x2(hh[k], mean, v[k]), dup(rh));
            rh = rsqrtf(fmaf(sum.y, inv_n, a.eps));
        }
        cl.write(static_cast<T*>(a.dh) + r * a.cols, v);
        if (r + 1 == group_end || !more) {
#pragma unroll
            for (int k = 0; k < kPairs; ++k) s_col[k] = mul_f32x2(s_col[k], dup(a.beta));
            if (wpost) {
                cl.weights(gate ? gate + group * a.cols : nullptr, w);
                if (!first_group) cl.read_f32(my_post, t);
#pragma unroll
                for (int k = 0; k < kPairs; ++k) w[k] = fma_f32x2(w[k], s_col[k], first_group ? 0 : t[k]);
                cl.write_f32(my_post, w);
            }
            if (gate) {  // the group is finished if it began in this range, else this is a partial sum
                const long long begin = group * a.group;
                cl.weights(wpost, w);
#pragma unroll
                for (int k = 0; k < kPairs; ++k) w[k] = mul_f32x2(w[k], s_col[k]);
                if (begin >= r0 && group_end <= r1) cl.write(static_cast<T*>(a.dgate) + group * a.cols, w);
                else cl.write_f32(my_gate + (begin < r0 ? 0 : a.part), w);
            }
#pragma unroll
            for (int k = 0; k < kPairs; ++k) s_col[k] = 0;
            first_group = false;
            ++group;
            group_end += a.group;
            if constexpr (KEEP) if (more) keep_factor();
        }
    }
    pdl_trigger();
    if (wpre) cl.write_f32(my_pre, s_pre);
    cp_wait(0);
}

// Adds the CTAs' partial sums.  Item 0 is w_post, 1 is w_pre, the others are gate
// groups: 2 + g is group g (by_border == 0), or 1 + c the group that the border
// between CTAs c - 1 and c is the first to cut, if there is one, so that there are at
// most as many items as groups and as borders.
struct SumArgs {
    const float *part_post, *part_pre, *part_gate;
    void *dw_post, *dw_pre, *dgate;
    long long per_cta, group;
    uint32_t cols, part;
    int ctas, items, by_border;
};

// A block adds LANES * 4 columns: each LANES threads every SEGS-th partial row, then the warps' sums, in a fixed order.
template <typename T, int LANES, int WARPS> __global__ void __launch_bounds__(32 * WARPS) norm_residual_sum_kernel(const SumArgs a) {
    constexpr int SEGS = WARPS * 32 / LANES, COLS = LANES * 4;
    __shared__ float4 part[WARPS][LANES];
    const int lane = threadIdx.x % LANES, seg = threadIdx.x / LANES;
    const uint32_t col = blockIdx.x * COLS + lane * 4;
    pdl_wait();
    for (int item = blockIdx.y; item < a.items; item += gridDim.y) {
        const float* src;
        T* dst;
        int c0 = 0, c1 = a.ctas;
        long long stride = a.part;
        if (item < 2) {
            src = item == 0 ? a.part_post : a.part_pre;
            dst = static_cast<T*>(item == 0 ? a.dw_post : a.dw_pre);
            if (!dst) continue;
        } else {
            const long long border = static_cast<long long>(item - 1) * a.per_cta;
            const long long g = a.by_border ? border / a.group : item - 2, begin = g * a.group;
            c0 = static_cast<int>(begin / a.per_cta);
            c1 = static_cast<int>((begin + a.group - 1) / a.per_cta) + 1;
            if (c1 - c0 == 1 || (a.by_border && c0 != item - 2)) continue;  // finished by its CTA, or not cut here first
            src = a.part_gate;
            dst = static_cast<T*>(a.dgate) + g * a.cols;
            stride *= 2;
        }
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
        if (col < a.cols) {
            const float* p = src + c0 * stride + col;
            // a group's first CTA keeps it in its second slot (it begins there), the later ones in their first
            const long long first = item >= 2 ? a.part : 0;
#pragma unroll 8
            for (int c = seg; c < c1 - c0; c += SEGS) {
                const float4 v = *reinterpret_cast<const float4*>(p + c * stride + (c == 0 ? first : 0));
                s.x += v.x;
                s.y += v.y;
                s.z += v.z;
                s.w += v.w;
            }
        }
#pragma unroll
        for (int d = LANES; d < 32; d *= 2) {
            s.x += __shfl_xor_sync(0xffffffffu, s.x, d);
            s.y += __shfl_xor_sync(0xffffffffu, s.y, d);
            s.z += __shfl_xor_sync(0xffffffffu, s.z, d);
            s.w += __shfl_xor_sync(0xffffffffu, s.w, d);
        }
        if ((threadIdx.x & 31) < LANES) part[threadIdx.x >> 5][lane] = s;
        __syncthreads();
        if (threadIdx.x < COLS && blockIdx.x * COLS + threadIdx.x < a.cols) {
            const float* column = reinterpret_cast<const float*>(part) + threadIdx.x;
            float t = 0.f;
#pragma unroll 8
            for (int w = 0; w < WARPS; ++w) t += column[w * COLS];
            dst[blockIdx.x * COLS + threadIdx.x] = Conv<T>::down(t);
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------- host side

constexpr int kRingBytes = 200 * 1024;  // shared memory of one SM given to rings

// Ring of a CTA when `per_sm` of them share an SM: up to 3 rows of `tensors`
// tensors beside `kept` bytes.  Returns the bytes of both.
int plan_ring(NormArgs& a, uint32_t pitch, int tensors, int kept, int per_sm) {
    a.pitch = pitch;
    const int slot = static_cast<int>(pitch) * tensors, fit = (kRingBytes / per_sm - kept) / slot;
    a.stages = fit < 1 ? 1 : fit > 3 ? 3 : static_cast<uint32_t>(fit);
    return slot * static_cast<int>(a.stages) + kept;
}

template <typename T, bool VEC, int THREADS> int launch_fwd(NormArgs a, cudaStream_t st) {
    constexpr int per_sm = THREADS == 32 ? 24 : 1024 / THREADS;
    const int smem = plan_ring(a, Cols<T, VEC, THREADS>::pitch(a.cols), 2, 0, per_sm);
    auto norm_kern = norm_residual_kernel<T, VEC, THREADS>;
    static SmemLimit limit;
    if (int rc = limit.ensure(norm_kern, smem, "norm_gate_residual")) return rc;
    const long long cap = static_cast<long long>(sm_count()) * per_sm;
    a.per_cta = (a.rows + cap - 1) / cap;
    launch_pdl(norm_kern, static_cast<unsigned>((a.rows + a.per_cta - 1) / a.per_cta), THREADS, static_cast<size_t>(smem), st, a);
    return launch_status("norm_gate_residual");
}

// The block with the fewest idle columns.  Without the blocks of 160 and 384 threads (bf16, cold caches, forward /
// backward): 16384 x 2560 79.9 / 131.7 us in 256 threads, 65.5 / 96.9 in 160; 8192 x 6144 84.0 / 148.1 us in 512,
// 77.8 / 127.6 in 384 (fp32 there 139.3 / 252.5 and 135.2 / 254.6).
template <typename T, bool VEC> int forward(const NormArgs& a, cudaStream_t st) {
    if (a.cols <= 32 * kEpt) return launch_fwd<T, VEC, 32>(a, st);
    if (a.cols <= 64 * kEpt) return launch_fwd<T, VEC, 64>(a, st);
    if (a.cols <= 96 * kEpt) return launch_fwd<T, VEC, 96>(a, st);
    if (a.cols <= 128 * kEpt) return launch_fwd<T, VEC, 128>(a, st);
    if (a.cols <= 160 * kEpt) return launch_fwd<T, VEC, 160>(a, st);
    if (a.cols <= 256 * kEpt) return launch_fwd<T, VEC, 256>(a, st);
    if (a.cols <= 320 * kEpt) return launch_fwd<T, VEC, 320>(a, st);
    if (a.cols <= 384 * kEpt) return launch_fwd<T, VEC, 384>(a, st);
    if (a.cols <= 512 * kEpt) return launch_fwd<T, VEC, 512>(a, st);
    if (sizeof(T) == 4 || a.cols <= 768 * kEpt) return launch_fwd<T, VEC, 768>(a, st);
    if constexpr (sizeof(T) == 2) return launch_fwd<T, VEC, 1024>(a, st);
    return fail(cudaErrorInvalidValue, "norm_gate_residual: %u columns", a.cols);  // refused before
}

struct NormGrads {
    void *dw_post, *dgate, *dw_pre;
};

template <typename T, bool VEC, int THREADS> int launch_bwd(NormArgs a, const NormGrads& g, cudaStream_t st) {
    int per_sm = THREADS == 32 ? 16 : THREADS <= 512 ? 512 / THREADS : 1;
    const uint32_t pitch = Cols<T, VEC, THREADS>::pitch(a.cols);
    const int kept = keep_vectors<T>(THREADS) ? static_cast<int>(pitch) + THREADS * kEpt * 4 : 0;
    int smem = plan_ring(a, pitch, 4, kept, per_sm);
    // fewer CTAs per SM where each can then copy a row ahead (8192 x 4096 fp32: 135 -> 130 us, 20000 x 1024: 96 -> 88);
    // unaligned rows have a barrier per row to hide instead (8192 x 4095 fp32: 174 us as is, 205 with fewer)
    while (VEC && per_sm > 1 && a.stages < 2) smem = plan_ring(a, pitch, 4, kept, --per_sm);
    auto norm_grad_kern = norm_residual_grad_kernel<T, VEC, THREADS>;
    static SmemLimit limit;
    if (int rc = limit.ensure(norm_grad_kern, smem, "norm_gate_residual_backward")) return rc;
    const long long cap = static_cast<long long>(sm_count()) * per_sm;
    a.per_cta = (a.rows + cap - 1) / cap;
    const long long ctas = (a.rows + a.per_cta - 1) / a.per_cta;
    a.part = (a.cols + 3) / 4 * 4;
    const size_t one = static_cast<size_t>(a.part) * static_cast<size_t>(ctas), bytes = one * 4 * sizeof(float);
    void* mem = nullptr;
    cudaError_t e = pool_malloc(&mem, bytes, st);
    if (e != cudaSuccess) return api_fail(e, "norm_gate_residual_backward: scratch of %zu bytes: %s", bytes, cudaGetErrorString(e));
    a.part_post = static_cast<float*>(mem);
    a.part_pre = a.part_post + one;
    a.part_gate = a.part_pre + one;
    launch_pdl(norm_grad_kern, static_cast<unsigned>(ctas), THREADS, static_cast<size_t>(smem), st, a);
    int rc = launch_status("norm_gate_residual_backward");
    if (rc == 0) {
        const long long groups = g.dgate ? a.rows / a.group : 0, borders = g.dgate ? ctas - 1 : 0;
        const bool by_border = borders < groups;
        const int items = 2 + static_cast<int>(by_border ? borders : groups);
        const SumArgs s{a.part_post, a.part_pre, a.part_gate, g.dw_post, g.dw_pre, g.dgate, a.per_cta, a.group, a.cols, a.part,
                        static_cast<int>(ctas), items, by_border ? 1 : 0};
        // Many partial rows come with few columns: blocks of 32 columns (a 128-byte line of a row) spread them over
        // the SMs (4099 x 1111 fp32, 684 partial rows: 35.7 us the whole call, 39.1 with 128 columns and 32 warps;
        // 65536 x 512 bf16 76.1 against 80.8).  The gate groups that CTAs cut are many items of a few partial rows,
        // for which wide blocks are faster (20000 x 1500 fp32, groups of 10: 186 us against 198).
        const dim3 wide((a.cols + 127) / 128, static_cast<unsigned>(items < 256 ? items : 256));
        if (ctas <= 256) launch_pdl(norm_residual_sum_kernel<T, 32, 8>, wide, 256, 0, st, s);
        else if (items > 8) launch_pdl(norm_residual_sum_kernel<T, 32, 32>, wide, 1024, 0, st, s);
        else launch_pdl(norm_residual_sum_kernel<T, 8, 16>, dim3((a.cols + 31) / 32, static_cast<unsigned>(items)), 512, 0, st, s);
        rc = launch_status("norm_gate_residual_backward (sums)");
    }
    const cudaError_t e2 = cudaFreeAsync(mem, st);
    if (rc == 0 && e2 != cudaSuccess) rc = api_fail(e2, "norm_gate_residual_backward: %s", cudaGetErrorString(e2));
    return rc;
}

template <typename T, bool VEC> int backward(const NormArgs& a, const NormGrads& g, cudaStream_t st) {
    if (a.cols <= 32 * kEpt) return launch_bwd<T, VEC, 32>(a, g, st);
    if (a.cols <= 64 * kEpt) return launch_bwd<T, VEC, 64>(a, g, st);
    if (a.cols <= 96 * kEpt) return launch_bwd<T, VEC, 96>(a, g, st);
    if (a.cols <= 128 * kEpt) return launch_bwd<T, VEC, 128>(a, g, st);
    if (a.cols <= 160 * kEpt) return launch_bwd<T, VEC, 160>(a, g, st);
    if (a.cols <= 256 * kEpt) return launch_bwd<T, VEC, 256>(a, g, st);
    if (a.cols <= 320 * kEpt) return launch_bwd<T, VEC, 320>(a, g, st);
    if (a.cols <= 384 * kEpt) return launch_bwd<T, VEC, 384>(a, g, st);
    if (a.cols <= 512 * kEpt) return launch_bwd<T, VEC, 512>(a, g, st);
    if (sizeof(T) == 4 || a.cols <= 768 * kEpt) return launch_bwd<T, VEC, 768>(a, g, st);
    if constexpr (sizeof(T) == 2) return launch_bwd<T, VEC, 1024>(a, g, st);
    return fail(cudaErrorInvalidValue, "norm_gate_residual: %u columns", a.cols);  // refused before
}

int check(const char* what, int dt, size_t rows, size_t cols, size_t group, bool gate, float alpha, float beta, float eps) {
    if (dt != DT_F32 && dt != DT_BF16 && dt != DT_F16) return fail(cudaErrorInvalidValue, "%s: unsupported dtype %d", what, dt);
    if (cols == 0 || cols > max_cols(dt)) return fail(cudaErrorInvalidValue, "%s: %zu columns outside [1, %zu]", what, cols, max_cols(dt));
    if (rows > (size_t{1} << 40)) return fail(cudaErrorInvalidValue, "%s: %zu rows", what, rows);
    if (gate && group != 0 && rows % group != 0)
        return fail(cudaErrorInvalidValue, "%s: %zu rows are not a multiple of the gate's group of %zu", what, rows, group);
    if (!(eps >= 0.f) || !std::isfinite(eps)) return fail(cudaErrorInvalidValue, "%s: eps must be finite and >= 0", what);
    if (!std::isfinite(alpha) || !std::isfinite(beta)) return fail(cudaErrorInvalidValue, "%s: alpha and beta must be finite", what);
    return 0;
}

// A tensor's bytes; an absent one has none.
struct Span {
    const void* p;
    size_t bytes;
    bool meets(const Span& o) const {
        const auto a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(o.p);
        return p && o.p && a < b + o.bytes && b < a + bytes;
    }
    bool crosses(const Span& o) const { return p != o.p && meets(o); }  // overlaps, and is not the same tensor
};

// Every given pointer is aligned to `to` bytes.
template <typename... P> bool aligned(uintptr_t to, const P*... p) { return (((reinterpret_cast<uintptr_t>(p)) | ...) & (to - 1)) == 0; }

}  // namespace

}  // namespace bee_b200

using namespace bee_b200;

extern "C" {

int bee_b200_norm_gate_residual(int dt, const void* h, const void* x, const void* w_post, const void* gate, const void* w_pre,
                                void* x_out, void* y, size_t rows, size_t cols, size_t group, float alpha, float beta,
                                float eps, bee_b200_stream_t stream) {
    const char* what = "norm_gate_residual";
    if (int rc = check(what, dt, rows, cols, group, gate != nullptr, alpha, beta, eps)) return rc;
    if (rows == 0) return ok();
    if (!h || !x || !x_out || (w_pre && !y)) return fail(cudaErrorInvalidValue, "%s: null pointer", what);
    const size_t elem = dt == DT_F32 ? 4 : 2;
    if (!aligned(elem, h, x, w_post, gate, w_pre, x_out, y))
        return fail(cudaErrorInvalidValue, "%s: a tensor is not aligned to its type", what);
    // rows are read ahead and by many CTAs: an output may take the place of h or x only row by row
    const size_t vector = cols * elem, tensor = rows * vector;
    const Span in[2] = {{h, tensor}, {x, tensor}}, out[2] = {{x_out, tensor}, {w_pre ? y : nullptr, tensor}};
    const Span vectors[3] = {{w_post, vector}, {gate, group ? rows / group * vector : vector}, {w_pre, vector}};
    bool apart = !out[0].meets(out[1]);
    for (const Span& o : out) {
        for (const Span& i : in) apart = apart && !o.crosses(i);
        for (const Span& v : vectors) apart = apart && !o.meets(v);
    }
    if (!apart) return fail(cudaErrorInvalidValue, "%s: outputs must not overlap each other, nor an input unless x_out or y is h or x", what);
    NormArgs a{};
    a.h = h; a.x = x; a.w_post = w_post; a.gate = gate; a.w_pre = w_pre; a.x_out = x_out; a.y = y;
    a.rows = static_cast<long long>(rows);
    a.group = static_cast<long long>(group ? group : rows);
    a.cols = static_cast<uint32_t>(cols);
    a.alpha = alpha; a.beta = beta; a.eps = eps;
    const bool vec = cols * elem % 16 == 0 && aligned(16, h, x, w_post, gate, w_pre, x_out, y);
    cudaStream_t st = as_stream(stream);
    if (dt == DT_F32) return vec ? forward<float, true>(a, st) : forward<float, false>(a, st);
    if (dt == DT_BF16) return vec ? forward<__nv_bfloat16, true>(a, st) : forward<__nv_bfloat16, false>(a, st);
    return vec ? forward<__half, true>(a, st) : forward<__half, false>(a, st);
}

int bee_b200_norm_gate_residual_backward(int dt, const void* h, const void* x, const void* w_post, const void* gate,
                                         const void* w_pre, const void* dx_out, const void* dy, void* dh, void* dx,
                                         void* dw_post, void* dgate, void* dw_pre, size_t rows, size_t cols, size_t group,
                                         float alpha, float beta, float eps, bee_b200_stream_t stream) {
    const char* what = "norm_gate_residual_backward";
    if (int rc = check(what, dt, rows, cols, group, gate != nullptr, alpha, beta, eps)) return rc;
    const size_t elem = dt == DT_F32 ? 4 : 2;
    if ((w_post && !dw_post) || (gate && !dgate) || (w_pre && !dw_pre)) return fail(cudaErrorInvalidValue, "%s: null pointer", what);
    cudaStream_t st = as_stream(stream);
    if (rows == 0) {  // sums over no rows (a gate per group has no rows either)
        cudaError_t e = cudaSuccess;
        if (w_post) e = cudaMemsetAsync(dw_post, 0, cols * elem, st);
        if (w_pre && e == cudaSuccess) e = cudaMemsetAsync(dw_pre, 0, cols * elem, st);
        if (gate && group == 0 && e == cudaSuccess) e = cudaMemsetAsync(dgate, 0, cols * elem, st);
        return e == cudaSuccess ? ok() : api_fail(e, "%s: %s", what, cudaGetErrorString(e));
    }
    if (!h || !x || !dh || !dx || (w_pre && !dy) || (!dx_out && !w_pre)) return fail(cudaErrorInvalidValue, "%s: null pointer", what);
    if (!aligned(elem, h, x, w_post, gate, w_pre, dx_out, dy, dh, dx, dw_post, dgate, dw_pre))
        return fail(cudaErrorInvalidValue, "%s: a tensor is not aligned to its type", what);
    // as in the forward; gate gradients are written while other rows are read, those of the weights after all of them
    const size_t vector = cols * elem, tensor = rows * vector, gates = group ? rows / group * vector : vector;
    const Span in[4] = {{h, tensor}, {x, tensor}, {dx_out, tensor}, {w_pre ? dy : nullptr, tensor}};
    const Span vectors[3] = {{w_post, vector}, {gate, gates}, {w_pre, vector}};
    const Span out[5] = {{dh, tensor}, {dx, tensor}, {gate ? dgate : nullptr, gates}, {w_post ? dw_post : nullptr, vector},
                         {w_pre ? dw_pre : nullptr, vector}};
    bool apart = true;
    for (int i = 0; i < 5; ++i)
        for (int j = 0; j < i; ++j) apart = apart && !out[i].meets(out[j]);
    for (int o = 0; o < 2; ++o) {
        for (const Span& i : in) apart = apart && !out[o].crosses(i);
        for (const Span& v : vectors) apart = apart && !out[o].meets(v);
    }
    for (const Span& i : in) apart = apart && !out[2].meets(i);
    apart = apart && !out[2].meets(vectors[0]) && !out[2].meets(vectors[2]) && !out[2].crosses(vectors[1]);
    if (!apart) return fail(cudaErrorInvalidValue, "%s: gradients must not overlap each other, nor an input unless dh or dx is one of its shape", what);
    NormArgs a{};
    a.h = h; a.x = x; a.w_post = w_post; a.gate = gate; a.w_pre = w_pre;
    a.dx_out = dx_out; a.dy = w_pre ? dy : nullptr; a.dh = dh; a.dx = dx; a.dgate = dgate;
    a.rows = static_cast<long long>(rows);
    a.group = static_cast<long long>(group ? group : rows);
    a.cols = static_cast<uint32_t>(cols);
    a.alpha = alpha; a.beta = beta; a.eps = eps;
    const NormGrads g{w_post ? dw_post : nullptr, gate ? dgate : nullptr, w_pre ? dw_pre : nullptr};
    const bool vec = cols * elem % 16 == 0 && aligned(16, h, x, w_post, gate, w_pre, dx_out, dy, dh, dx, gate ? dgate : nullptr);
    if (dt == DT_F32) return vec ? backward<float, true>(a, g, st) : backward<float, false>(a, g, st);
    if (dt == DT_BF16) return vec ? backward<__nv_bfloat16, true>(a, g, st) : backward<__nv_bfloat16, false>(a, g, st);
    return vec ? backward<__half, true>(a, g, st) : backward<__half, false>(a, g, st);
}

}  // extern "C"
