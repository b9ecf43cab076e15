// The first half of a gated feed-forward block, out = act(x Wg) * (x Wu), and
// its gradient, for 16-bit tensors with fp32 accumulation.  New: the reference
// has no such block; bmm and elementwise ops are the unfused form.
//
// Forward, many rows: both products in one kernel.  Two CTAs of a cluster
// compute a 256-row tile of 128 columns of both with one tcgen05.mma
// (cta_group::2, M = 256, N = 256) per K step: the leader loads 128 columns of
// Wg, its peer the same columns of Wu, and the accumulator's halves are g and u
// of the same outputs, so that the epilogue forms act(g) u from its own lanes.
//
// Forward, up to 64 rows (serving): bound by reading the weights once.  The
// weights are the M operand (128 of their columns per CTA, for g and for u) and
// the rows of x the N operand, padded only to 16, 32 or 64.  Where the
// columns give too few CTAs, a cluster cuts K and joins its partial sums, in
// rank order, through distributed shared memory.
//
// Backward, from x, the weights, the g and u that the forward kept, and dout:
//   du = dout act(g), dg = dout u act'(g)     one elementwise pass, rounded to 16 bits
//                                             (the tensor cores' operand type)
//   dx = dg Wg^T + du Wu^T                    one product, K running over both halves
//   dWg = x^T dg, dWu = x^T du                one launch, both operands MN-major
// Bound by the tensor cores: 4 M D F flops forward and 8 M D F backward.
//
// TMA needs 16-byte row strides: operands whose rows are not (odd sizes, odd
// slices) are first copied to padded scratch.  Every mbarrier wait is bounded and
// reports through bee_b200_device_status.
#include <cmath>

#include "common.cuh"
#include "sm100.cuh"
#include "tc_tiles.cuh"

namespace bee_b200 {

using namespace sm100;

namespace {

// Device status word: code of the first bounded wait that gave up (0 = none).
__device__ int g_gated_status = 0;

enum Act : int { ACT_SILU = 0, ACT_GELU = 1, ACT_GELU_TANH = 2 };

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kTanhC = 0.7978845608028654f;  // sqrt(2 / pi)
constexpr float kTanhA = 0.044715f;

__device__ __forceinline__ float sigmoid(float v) { return __fdividef(1.f, 1.f + exp2f(-v * kLog2e)); }

// gelu (tanh) is g * sigmoid(2 c (g + a g^3)), since (1 + tanh z) / 2 = sigmoid(2 z).
__device__ __forceinline__ float activation(float g, int act) {
    if (act == ACT_SILU) return g * sigmoid(g);
    if (act == ACT_GELU) return g * normcdff(g);
    return g * sigmoid(2.f * kTanhC * fmaf(kTanhA * g * g, g, g));
}

// The activation and its derivative.  The factors of p = sigmoid or Phi that grow with g take a clamped g, so that
// they stay finite where p is 0 or 1 to the last bit and the derivative with it: past |g| = 88 for silu, whose p is
// still e^g below it, and past 32 for the gelus.
__device__ __forceinline__ void activation_grad(float g, int act, float& a, float& da) {
    if (act == ACT_SILU) {
        const float p = sigmoid(g);
        a = g * p;
        da = p * fmaf(fminf(fmaxf(g, -128.f), 128.f), 1.f - p, 1.f);
        return;
    }
    const float c = fminf(fmaxf(g, -32.f), 32.f);
    if (act == ACT_GELU) {
        const float p = normcdff(g);
        a = g * p;
        da = fmaf(c * 0.3989422804014327f, exp2f(-0.5f * kLog2e * c * c), p);
    } else {
        const float p = sigmoid(2.f * kTanhC * fmaf(kTanhA * g * g, g, g));
        a = g * p;
        const float z = kTanhC * fmaf(3.f * kTanhA * c, c, 1.f);
        da = p * fmaf(2.f * c * z, 1.f - p, 1.f);
    }
}

// g = act(g) u for N columns in registers (bits of fp32).  One loop per activation: with the choice inside, the
// unrolled code of all three outgrows the instruction cache (1024 x 1024 -> 4096: 47 us against 25).
template <int N> __device__ __forceinline__ void gate_columns(uint32_t (&g)[N], const uint32_t (&u)[N], int act) {
    if (act == ACT_SILU) {
#pragma unroll
        for (int j = 0; j < N; ++j) g[j] = __float_as_uint(activation(__uint_as_float(g[j]), ACT_SILU) * __uint_as_float(u[j]));
    } else if (act == ACT_GELU) {
#pragma unroll
        for (int j = 0; j < N; ++j) g[j] = __float_as_uint(activation(__uint_as_float(g[j]), ACT_GELU) * __uint_as_float(u[j]));
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) g[j] = __float_as_uint(activation(__uint_as_float(g[j]), ACT_GELU_TANH) * __uint_as_float(u[j]));
    }
}

__device__ __forceinline__ uint32_t pack16(float lo, float hi, int f16) { return f16 ? pack_f16x2(lo, hi) : pack_bf16x2(lo, hi); }
__device__ __forceinline__ uint16_t round16(float v, int f16) { return static_cast<uint16_t>(pack16(v, 0.f, f16) & 0xffffu); }
__device__ __forceinline__ float up16(uint16_t v, int f16) {
    return f16 ? __half2float(__ushort_as_half(v)) : __uint_as_float(static_cast<uint32_t>(v) << 16);
}

// 32 consecutive columns of one output row, the first n of them inside it.
__device__ __forceinline__ void store32(uint16_t* dst, const float (&v)[32], int n, int vec, int f16) {
    if (n >= 32 && vec) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            reinterpret_cast<uint4*>(dst)[j] = make_uint4(pack16(v[8 * j], v[8 * j + 1], f16), pack16(v[8 * j + 2], v[8 * j + 3], f16),
                                                          pack16(v[8 * j + 4], v[8 * j + 5], f16), pack16(v[8 * j + 6], v[8 * j + 7], f16));
    } else {
#pragma unroll
        for (int j = 0; j < 32; ++j)
            if (j < n) dst[j] = round16(v[j], f16);
    }
}

// ---------------------------------------------------------------- CTA-pair products

enum Mode : int {
    FORWARD,  // A = x; rank 0 loads Wg, rank 1 Wu; epilogue act(g) u
    DX,       // A = dg then du, B = Wg then Wu along K
    DW,       // A = x^T or dg^T / du^T, B the other one; the first tiles are dWg, the rest dWu
};

struct PairParams {
    int M, N;              // rows and columns of an output (FORWARD: columns of out)
    int m_tiles, n_tiles, tiles;  // tiles: of one output
    // Work items: `whole` tiles, then the remaining tiles, too few for one each per CTA pair, cut along K into
    // `cuts` items each, whose fp32 sums go to part[item][column / 4][row] for a second kernel to join in order.
    int items, whole, cuts;
    float4* part;
    int num_kb, half_kb;   // K blocks in all, and of the first half (DX)
    long long ldc;
    uint16_t* out[3];      // FORWARD: out, g, u (the last two may be null); DX: dx; DW: dWg, dWu
    int vec, f16, act;
    int a_second;          // DW: which operand differs between dWg and dWu (1: A, 0: B)
};

struct PairItem {
    int which, mb, nb;  // the output, and its tile
    int kb0, kbs;       // first K block and number of them
    int part;           // index of the partial sum, -1 for a whole tile
};

// First K block (or end, for cut + 1) of a cut tile's part.
__device__ __forceinline__ int cut_begin(const PairParams& p, int cut) {
    return static_cast<int>(static_cast<long long>(p.num_kb) * cut / p.cuts);
}

template <int MODE> __device__ __forceinline__ PairItem pair_item(const PairParams& p, int item) {
    PairItem w;
    int tile = item;
    w.kb0 = 0;
    w.kbs = p.num_kb;
    w.part = -1;
    if (item >= p.whole) {
        w.part = item - p.whole;
        tile = p.whole + w.part / p.cuts;
        const int cut = w.part % p.cuts;
        w.kb0 = cut_begin(p, cut);
        w.kbs = cut_begin(p, cut + 1) - w.kb0;
    }
    w.which = MODE == DW ? tile / p.tiles : 0;
    grouped_tile(tile - w.which * p.tiles, p.m_tiles, p.n_tiles, w.mb, w.nb);
    return w;
}

// Columns c * 32 to c * 32 + 31 of a tile's row (FORWARD: rg of g and ru of u, else rg alone), to the outputs.
template <int MODE>
__device__ __forceinline__ void store_tile_row(const PairParams& p, const PairItem& w, int row, int c, uint32_t (&rg)[32],
                                               const uint32_t (&ru)[32]) {
    constexpr int WIDTH = MODE == FORWARD ? 128 : 256;
    const int col = w.nb * WIDTH + c * 32, n = p.N - col;
    if (row >= p.M || n <= 0) return;
    const long long o = static_cast<long long>(row) * p.ldc + col;
    float v[32];
    if constexpr (MODE == FORWARD) {
        if (p.out[1]) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(rg[j]);
            store32(p.out[1] + o, v, n, p.vec, p.f16);
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(ru[j]);
            store32(p.out[2] + o, v, n, p.vec, p.f16);
        }
        gate_columns(rg, ru, p.act);
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(rg[j]);
        store32(p.out[0] + o, v, n, p.vec, p.f16);
    } else {
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(rg[j]);
        store32((MODE == DW && w.which ? p.out[1] : p.out[0]) + o, v, n, p.vec, p.f16);
    }
}

// 256 x 256 accumulators (FORWARD: 128 columns of g and 128 of u), BK = 128 per
// stage in boxes of 16 KiB, three stages; two accumulators in TMEM so that a
// tile's epilogue overlaps the next tile's products.
struct PairCfg {
    static constexpr int BM = 256, BN = 256, BK = 128;
    static constexpr int BOX = 128 * 64 * 2;
    static constexpr int STAGE = 4 * BOX;  // this CTA's 128 rows of A and 128 columns of B
    static constexpr int STAGES = 3;
    static constexpr int OUT = 32 * 64 * 2;  // an epilogue warp's 32 rows of 64 output columns, as TMA stores them
    static constexpr int SMEM = STAGES * STAGE + 4 * 2 * OUT + 1024;
    static constexpr uint32_t TMEM_COLS = 512;
};

// One epilogue warp's 32 rows x 64 columns: rounded into its next staging buffer (128-byte rows, swizzled as the map
// says) and stored by TMA, which cuts what lies outside the output in whole 16-byte blocks only; outputs whose strides
// or columns are no whole number of those are written from the buffer row by row, a column per lane.  v(j): the lane's row's column j.
template <typename V>
__device__ __forceinline__ void store_block(const PairParams& p, const CUtensorMap* map, uint16_t* out, uint8_t* stage, int& turn, int lane,
                                            int row0, int col, V v) {
    if (lane == 0) tma_store_wait_read_all_but<1>();  // the buffer's last store has been read
    __syncwarp();
    uint8_t* block = stage + turn * PairCfg::OUT;
#pragma unroll
    for (int c = 0; c < 8; ++c)
        *reinterpret_cast<uint4*>(block + lane * 128 + ((c ^ (lane & 7)) << 4)) =
            make_uint4(pack16(v(8 * c), v(8 * c + 1), p.f16), pack16(v(8 * c + 2), v(8 * c + 3), p.f16),
                       pack16(v(8 * c + 4), v(8 * c + 5), p.f16), pack16(v(8 * c + 6), v(8 * c + 7), p.f16));
    if (p.vec) {
        fence_async_smem();
        __syncwarp();
        if (lane == 0) {
            tma_store_3d(map, block, col, row0, 0);
            tma_store_commit();
        }
    } else {
        __syncwarp();
        const int rows = min(32, p.M - row0);
        for (int r = 0; r < rows; ++r) {
            uint16_t* dst = out + static_cast<long long>(row0 + r) * p.ldc + col;
#pragma unroll
            for (int j = lane; j < 64; j += 32) {
                const uint16_t x = *reinterpret_cast<const uint16_t*>(block + r * 128 + (((j >> 3) ^ (r & 7)) << 4) + (j & 7) * 2);
                if (col + j < p.N) dst[j] = x;
            }
        }
    }
    turn ^= 1;
}

template <int MODE, bool A_MN, bool B_MN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(192, 1)
    gated_pair_kernel(const __grid_constant__ CUtensorMap tmA0, const __grid_constant__ CUtensorMap tmA1,
                      const __grid_constant__ CUtensorMap tmB0, const __grid_constant__ CUtensorMap tmB1,
                      const __grid_constant__ CUtensorMap tmO0, const __grid_constant__ CUtensorMap tmO1,
                      const __grid_constant__ CUtensorMap tmO2, const PairParams p) {
    using Cfg = PairCfg;
    constexpr int STAGES = Cfg::STAGES;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[STAGES];
    __shared__ __align__(8) uint64_t empty_bar[STAGES];
    __shared__ __align__(8) uint64_t tfull_bar[2];
    __shared__ __align__(8) uint64_t tempty_bar[2];
    __shared__ __align__(8) uint64_t done_bar;
    __shared__ uint32_t tmem_base_sh;
    __shared__ int abort_sh;

    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    volatile int* abort_flag = &abort_sh;
    int* status = &g_gated_status;
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();  // 0 = leader
    const bool leader = rank == 0;
    const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(&tfull_bar[a], 1);
            mbar_init(&tempty_bar[a], 8);  // 4 epilogue warps in each CTA of the pair
        }
        mbar_init(&done_bar, 1);
        abort_sh = 0;
        fence_mbar_init();
    }
    if (warp == 0 && lane == 0) {
        tma_prefetch(&tmA0);
        tma_prefetch(&tmB0);
        if (MODE != FORWARD) tma_prefetch(&tmA1);
        tma_prefetch(&tmB1);
    }
    if (warp == 1) tmem_alloc_pair<Cfg::TMEM_COLS>(&tmem_base_sh);
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // both CTAs' barriers and TMEM exist before any cross-CTA traffic
    tc_fence_after();
    const uint32_t tmem_base = tmem_base_sh;

    if (warp == 0) {
        // ------------------------------------------------ TMA producer (both CTAs)
        int stage = 0;
        uint32_t phase = 0;
        long long issued = 0;
        for (int item = pair; item < p.items; item += npairs) {
            if (__any_sync(0xffffffffu, *abort_flag != 0)) break;
            const PairItem w = pair_item<MODE>(p, item);
            for (int kb = 0; kb < w.kbs; ++kb) {
                bool ok = true;
                if (lane == 0) ok = mbar_wait(&empty_bar[stage], phase ^ 1u, abort_flag, status, 31);
                ok = __shfl_sync(0xffffffffu, ok, 0);
                if (!ok) break;
                if (lane == 0) {
                    uint8_t* sa = smem + stage * Cfg::STAGE;
                    uint8_t* sb = sa + 2 * Cfg::BOX;
                    const uint32_t full_leader = mapa_shared(smem_u32(&full_bar[stage]), 0);
                    if (leader) mbar_arrive_expect_tx(&full_bar[stage], 2 * Cfg::STAGE);
                    int k = w.kb0 + k_block(kb, item / npairs, w.kbs);
                    bool second_a = false, second_b = false;
                    if (MODE == FORWARD) {
                        second_b = !leader;
                    } else if (MODE == DX) {
                        second_a = second_b = k >= p.half_kb;
                        if (second_a) k -= p.half_kb;
                    } else {
                        second_a = w.which != 0 && p.a_second;
                        second_b = w.which != 0 && !p.a_second;
                    }
                    const CUtensorMap* ta = second_a ? &tmA1 : &tmA0;
                    const CUtensorMap* tb = second_b ? &tmB1 : &tmB0;
                    const int m0 = w.mb * Cfg::BM + static_cast<int>(rank) * 128;
                    const int n0 = MODE == FORWARD ? w.nb * 128 : w.nb * Cfg::BN + static_cast<int>(rank) * 128;
                    const int k0 = k * Cfg::BK;
                    if constexpr (A_MN) {
                        tma_load_3d_pair(sa, ta, full_leader, m0, k0, 0);
                        tma_load_3d_pair(sa + Cfg::BOX, ta, full_leader, m0 + 64, k0, 0);
                    } else {
                        tma_load_3d_pair(sa, ta, full_leader, k0, m0, 0);
                        tma_load_3d_pair(sa + Cfg::BOX, ta, full_leader, k0 + 64, m0, 0);
                    }
                    if constexpr (B_MN) {
                        tma_load_3d_pair(sb, tb, full_leader, n0, k0, 0);
                        tma_load_3d_pair(sb + Cfg::BOX, tb, full_leader, n0 + 64, k0, 0);
                    } else {
                        tma_load_3d_pair(sb, tb, full_leader, k0, n0, 0);
                        tma_load_3d_pair(sb + Cfg::BOX, tb, full_leader, k0 + 64, n0, 0);
                    }
                }
                __syncwarp();
                ++issued;
                if (++stage == STAGES) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
        }
        // Drain: the leader's full barriers count both CTAs' loads; the last of
        // them must have landed before the final cluster barrier lets a CTA exit.
        if (lane == 0 && leader) {
            const long long first = issued > STAGES ? issued - STAGES : 0;
            for (long long it = first; it < issued; ++it)
                mbar_wait(&full_bar[it % STAGES], static_cast<uint32_t>((it / STAGES) & 1), abort_flag, status, 32, 200000000ull);
        }
        __syncwarp();
    } else if (warp == 1) {
        // ------------------------------------------------ MMA issuer (leader CTA only)
        if (leader) {
            const uint32_t idesc = idesc_f16_f32(256, 256, A_MN, B_MN, p.f16 != 0);
            int stage = 0;
            uint32_t phase = 0;
            int local = 0;
            bool issued_any = false;
            for (int item = pair; item < p.items; item += npairs, ++local) {
                if (__any_sync(0xffffffffu, *abort_flag != 0)) break;
                const int cut = item < p.whole ? 0 : (item - p.whole) % p.cuts;
                const int kbs = item < p.whole ? p.num_kb : cut_begin(p, cut + 1) - cut_begin(p, cut);
                const int acc = local & 1;
                const uint32_t acc_phase = static_cast<uint32_t>((local >> 1) & 1);
                bool ok = true;
                if (lane == 0) ok = mbar_wait_cluster(&tempty_bar[acc], acc_phase ^ 1u, abort_flag, status, 33);
                ok = __shfl_sync(0xffffffffu, ok, 0);
                if (!ok) break;
                tc_fence_after();
                const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * Cfg::BN);
                for (int kb = 0; kb < kbs; ++kb) {
                    if (lane == 0) ok = mbar_wait(&full_bar[stage], phase, abort_flag, status, 34);
                    ok = __shfl_sync(0xffffffffu, ok, 0);
                    if (!ok) break;
                    tc_fence_after();
                    if (lane == 0) {
                        const uint32_t a_base = smem_u32(smem + stage * Cfg::STAGE);
                        const uint32_t b_base = a_base + 2 * Cfg::BOX;
#pragma unroll
                        for (int k = 0; k < Cfg::BK / 16; ++k) {
                            // K-major: two 64-wide K halves of 16 KiB, 32 bytes per 16-K step in a half;
                            // MN-major: two 64-wide MN chunks of 16 KiB, 128 bytes per K row
                            const uint32_t kmaj = (k / 4) * Cfg::BOX + (k % 4) * 32;
                            const uint64_t adesc = A_MN ? sdesc_sw128(a_base + k * 16 * 128, Cfg::BOX, 1024) : sdesc_sw128(a_base + kmaj, 16, 1024);
                            const uint64_t bdesc = B_MN ? sdesc_sw128(b_base + k * 16 * 128, Cfg::BOX, 1024) : sdesc_sw128(b_base + kmaj, 16, 1024);
                            mma_f16_ss_pair(d_tmem, adesc, bdesc, idesc, (kb | k) != 0 ? 1u : 0u);
                        }
                        mma_commit_pair(&empty_bar[stage], 0x3);
                        issued_any = true;
                    }
                    __syncwarp();
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                if (!ok) break;
                if (lane == 0) mma_commit_pair(&tfull_bar[acc], 0x3);
                __syncwarp();
            }
            if (lane == 0 && issued_any) {
                mma_commit_pair(&done_bar, 0x1);
                mbar_wait(&done_bar, 0, abort_flag, status, 35, 200000000ull);
            }
            __syncwarp();
        }
    } else {
        // ------------------------------------------------ epilogue (warps 2-5, both CTAs)
        const int q = warp & 3;
        const uint32_t tempty_leader0 = mapa_shared(smem_u32(&tempty_bar[0]), 0);
        const uint32_t tempty_leader1 = mapa_shared(smem_u32(&tempty_bar[1]), 0);
        uint8_t* out_stage = smem + STAGES * Cfg::STAGE + q * 2 * Cfg::OUT;
        int out_turn = 0;
        int local = 0;
        for (int item = pair; item < p.items; item += npairs, ++local) {
            if (__any_sync(0xffffffffu, *abort_flag != 0)) break;
            const PairItem w = pair_item<MODE>(p, item);
            const int acc = local & 1;
            const uint32_t acc_phase = static_cast<uint32_t>((local >> 1) & 1);
            bool ok = mbar_wait(&tfull_bar[acc], acc_phase, abort_flag, status, 36);
            if (!__all_sync(0xffffffffu, ok)) break;
            tc_fence_after();
            const int tile_row = static_cast<int>(rank) * 128 + q * 32 + lane;
            const uint32_t taddr = tmem_base + static_cast<uint32_t>(acc * Cfg::BN) + (static_cast<uint32_t>(q * 32) << 16);
            constexpr int STEP = MODE == FORWARD ? 128 : Cfg::BN;  // FORWARD: u is 128 columns after g
            const int row0 = w.mb * Cfg::BM + tile_row - lane;
            if (w.part < 0) {
#pragma unroll 1
                for (int c = 0; c < STEP; c += 64) {
                    uint32_t g0[32], g1[32], u0[32], u1[32];
                    tmem_ld_32x32b_x32(taddr + c, g0);
                    tmem_ld_32x32b_x32(taddr + c + 32, g1);
                    if (MODE == FORWARD) {
                        tmem_ld_32x32b_x32(taddr + 128 + c, u0);
                        tmem_ld_32x32b_x32(taddr + 128 + c + 32, u1);
                    }
                    tmem_ld_wait();
                    const int col = w.nb * STEP + c;
                    if (row0 < p.M && col < p.N) {
                        auto g = [&](int j) { return __uint_as_float(j < 32 ? g0[j & 31] : g1[j & 31]); };
                        auto u = [&](int j) { return __uint_as_float(j < 32 ? u0[j & 31] : u1[j & 31]); };
                        if constexpr (MODE == FORWARD) {
                            if (p.out[1]) {
                                store_block(p, &tmO1, p.out[1], out_stage, out_turn, lane, row0, col, g);
                                store_block(p, &tmO2, p.out[2], out_stage, out_turn, lane, row0, col, u);
                            }
                            gate_columns(g0, u0, p.act);
                            gate_columns(g1, u1, p.act);
                            store_block(p, &tmO0, p.out[0], out_stage, out_turn, lane, row0, col, g);
                        } else {
                            const bool second = MODE == DW && w.which;
                            store_block(p, second ? &tmO1 : &tmO0, second ? p.out[1] : p.out[0], out_stage, out_turn, lane, row0, col, g);
                        }
                    }
                    __syncwarp();  // the next TMEM load is a warp-wide instruction
                }
            } else {
                float4* part = p.part + static_cast<size_t>(w.part) * (Cfg::BM * Cfg::BN / 4) + tile_row;
#pragma unroll 1
                for (int c = 0; c < Cfg::BN / 32; ++c) {
                    uint32_t r[32];
                    tmem_ld_32x32b_x32(taddr + c * 32, r);
                    tmem_ld_wait();
#pragma unroll
                    for (int v = 0; v < 8; ++v)
                        part[(c * 8 + v) * Cfg::BM] = make_float4(__uint_as_float(r[4 * v]), __uint_as_float(r[4 * v + 1]),
                                                                  __uint_as_float(r[4 * v + 2]), __uint_as_float(r[4 * v + 3]));
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(acc ? tempty_leader1 : tempty_leader0);
        }
        if (lane == 0) tma_store_wait_read();  // the staging buffers must outlive their stores
        __syncwarp();
    }

    tc_fence_before();
    __syncthreads();
    cluster_sync();  // no CTA leaves while its peer may still touch its barriers or shared memory
    tc_fence_after();
    if (warp == 1) tmem_dealloc_pair<Cfg::TMEM_COLS>(tmem_base);
}

// Joins the cut tiles: block (t, c) adds the partial sums of columns c * 32 to c * 32 + 31
// (FORWARD: of g and of u) of tile `whole` + t, a row per thread, and stores the results.
template <int MODE> __global__ void __launch_bounds__(256) gated_pair_join_kernel(const PairParams p) {
    pdl_wait();
    const int first = blockIdx.x * p.cuts, c = blockIdx.y;
    const PairItem w = pair_item<MODE>(p, p.whole + first);
    uint32_t rg[32], ru[32];
    float4 g[8], u[8];
#pragma unroll
    for (int v = 0; v < 8; ++v) g[v] = u[v] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i = 0; i < p.cuts; ++i) {
        const float4* part = p.part + static_cast<size_t>(first + i) * (PairCfg::BM * PairCfg::BN / 4) + threadIdx.x;
#pragma unroll
        for (int v = 0; v < 8; ++v) {
            const float4 a = part[(c * 8 + v) * PairCfg::BM];
            g[v].x += a.x; g[v].y += a.y; g[v].z += a.z; g[v].w += a.w;
            if (MODE == FORWARD) {
                const float4 b = part[(32 + c * 8 + v) * PairCfg::BM];
                u[v].x += b.x; u[v].y += b.y; u[v].z += b.z; u[v].w += b.w;
            }
        }
    }
#pragma unroll
    for (int v = 0; v < 8; ++v) {
        rg[4 * v] = __float_as_uint(g[v].x); rg[4 * v + 1] = __float_as_uint(g[v].y);
        rg[4 * v + 2] = __float_as_uint(g[v].z); rg[4 * v + 3] = __float_as_uint(g[v].w);
        ru[4 * v] = __float_as_uint(u[v].x); ru[4 * v + 1] = __float_as_uint(u[v].y);
        ru[4 * v + 2] = __float_as_uint(u[v].z); ru[4 * v + 3] = __float_as_uint(u[v].w);
    }
    store_tile_row<MODE>(p, w, w.mb * PairCfg::BM + static_cast<int>(threadIdx.x), c, rg, ru);
}

// ---------------------------------------------------------------- few rows

struct RowsParams {
    int M, N;          // rows of x, columns of out
    int num_kb;        // 64-wide K blocks
    int cluster, stages;
    uint16_t* out[3];  // out, g, u
    int f16, act;
};

// One CTA: 128 columns of g and of u for all M <= NT rows, over its share of K.
template <int NT, bool W_MN>
__global__ void __launch_bounds__(192) gated_rows_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmG,
                                                         const __grid_constant__ CUtensorMap tmU, const RowsParams p) {
    constexpr int BK = 64, W_BYTES = 128 * BK * 2, X_BYTES = NT * BK * 2, STAGE = 2 * W_BYTES + X_BYTES;
    constexpr int MAX_STAGES = 6;
    constexpr uint32_t TMEM_COLS = 2 * NT;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[MAX_STAGES];
    __shared__ __align__(8) uint64_t empty_bar[MAX_STAGES];
    __shared__ __align__(8) uint64_t tfull_bar;
    __shared__ uint32_t tmem_base_sh;
    __shared__ int abort_sh;

    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    volatile int* abort_flag = &abort_sh;
    int* status = &g_gated_status;
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int rank = p.cluster > 1 ? static_cast<int>(cluster_ctarank()) : 0;
    const int f0 = (blockIdx.x / p.cluster) * 128;
    const int kb0 = static_cast<int>(static_cast<long long>(p.num_kb) * rank / p.cluster);
    const int kb1 = static_cast<int>(static_cast<long long>(p.num_kb) * (rank + 1) / p.cluster);

    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], 1);
        }
        mbar_init(&tfull_bar, 1);
        abort_sh = 0;
        fence_mbar_init();
    }
    if (warp == 0 && lane == 0) {
        tma_prefetch(&tmX);
        tma_prefetch(&tmG);
        tma_prefetch(&tmU);
    }
    if (warp == 1) tmem_alloc<TMEM_COLS>(&tmem_base_sh);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = tmem_base_sh;
    pdl_wait();
    pdl_trigger();

    if (warp == 0) {
        // ------------------------------------------------ TMA producer
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        int kb = kb0;
        for (; kb < kb1; ++kb) {
            if (lane == 0) ok = mbar_wait(&empty_bar[stage], phase ^ 1u, abort_flag, status, 41);
            ok = __shfl_sync(0xffffffffu, ok, 0);
            if (!ok) break;
            if (lane == 0) {
                uint8_t* sg = smem + stage * STAGE;
                uint8_t* su = sg + W_BYTES;
                uint8_t* sx = su + W_BYTES;
                mbar_arrive_expect_tx(&full_bar[stage], STAGE);
                if constexpr (W_MN) {
                    tma_load_3d(sg, &tmG, &full_bar[stage], f0, kb * BK, 0);
                    tma_load_3d(sg + W_BYTES / 2, &tmG, &full_bar[stage], f0 + 64, kb * BK, 0);
                    tma_load_3d(su, &tmU, &full_bar[stage], f0, kb * BK, 0);
                    tma_load_3d(su + W_BYTES / 2, &tmU, &full_bar[stage], f0 + 64, kb * BK, 0);
                } else {
                    tma_load_3d(sg, &tmG, &full_bar[stage], kb * BK, f0, 0);
                    tma_load_3d(su, &tmU, &full_bar[stage], kb * BK, f0, 0);
                }
                tma_load_3d(sx, &tmX, &full_bar[stage], kb * BK, 0, 0);
            }
            __syncwarp();
            if (++stage == p.stages) {
                stage = 0;
                phase ^= 1u;
            }
        }
        // after an abort the loads in flight must land before the CTA exits
        if (lane == 0) {
            const int issued = kb - kb0, first = issued > p.stages ? issued - p.stages : 0;
            for (int it = first; it < issued; ++it)
                mbar_wait(&full_bar[it % p.stages], static_cast<uint32_t>((it / p.stages) & 1), abort_flag, status, 42, 200000000ull);
        }
        __syncwarp();
    } else if (warp == 1) {
        // ------------------------------------------------ MMA issuer
        const uint32_t idesc = idesc_f16_f32(128, NT, W_MN, false, p.f16 != 0);
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int kb = kb0; kb < kb1; ++kb) {
            if (lane == 0) ok = mbar_wait(&full_bar[stage], phase, abort_flag, status, 43);
            ok = __shfl_sync(0xffffffffu, ok, 0);
            if (!ok) break;
            tc_fence_after();
            if (lane == 0) {
                const uint32_t g_base = smem_u32(smem + stage * STAGE);
                const uint32_t x_base = g_base + 2 * W_BYTES;
#pragma unroll
                for (int k = 0; k < BK / 16; ++k) {
                    const uint64_t xdesc = sdesc_sw128(x_base + k * 32, 16, 1024);
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
                        const uint32_t base = g_base + w * W_BYTES;
                        const uint64_t wdesc = W_MN ? sdesc_sw128(base + k * 16 * 128, W_BYTES / 2, 1024) : sdesc_sw128(base + k * 32, 16, 1024);
                        mma_f16_ss(tmem_base + w * NT, wdesc, xdesc, idesc, kb > kb0 || k != 0 ? 1u : 0u);
                    }
                }
                mma_commit(&empty_bar[stage]);
            }
            __syncwarp();
            if (++stage == p.stages) {
                stage = 0;
                phase ^= 1u;
            }
        }
        // completes when every product above has; waited for here too, so that TMEM is idle when it is freed
        if (lane == 0) {
            mma_commit(&tfull_bar);
            mbar_wait(&tfull_bar, 0, abort_flag, status, 44, 200000000ull);
        }
        __syncwarp();
    } else {
        // ------------------------------------------------ partial sums to shared memory: [2 * NT][128] floats
        // (the ring's memory: all its loads have been consumed when the products are complete)
        const bool ok = mbar_wait(&tfull_bar, 0, abort_flag, status, 45);
        if (__all_sync(0xffffffffu, ok)) {
            tc_fence_after();
            const int q = warp & 3;
            float* part = reinterpret_cast<float*>(smem);
#pragma unroll 1
            for (int c = 0; c < 2 * NT / 32; ++c) {
                uint32_t r[32];
                tmem_ld_32x32b_x32(tmem_base + c * 32 + (static_cast<uint32_t>(q * 32) << 16), r);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 32; ++j) part[(c * 32 + j) * 128 + q * 32 + lane] = __uint_as_float(r[j]);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (p.cluster > 1) cluster_sync();
    tc_fence_after();
    if (warp == 1) tmem_dealloc<TMEM_COLS>(tmem_base);

    // act(g) u for this CTA's share of the tile's outputs, row by row of x
    const uint32_t part0 = smem_u32(smem);
    for (int i = rank * 192 + static_cast<int>(threadIdx.x); i < p.M * 128; i += p.cluster * 192) {
        const int m = i >> 7, f = i & 127;
        if (f0 + f >= p.N) continue;
        float g = 0.f, u = 0.f;
        for (int s = 0; s < p.cluster; ++s) {
            const uint32_t base = p.cluster > 1 ? mapa_shared(part0, static_cast<uint32_t>(s)) : part0;
            float vg, vu;
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(vg) : "r"(base + (m * 128 + f) * 4) : "memory");
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(vu) : "r"(base + ((NT + m) * 128 + f) * 4) : "memory");
            g += vg;
            u += vu;
        }
        const long long o = static_cast<long long>(m) * p.N + f0 + f;
        if (p.out[1]) {
            p.out[1][o] = round16(g, p.f16);
            p.out[2][o] = round16(u, p.f16);
        }
        p.out[0][o] = round16(activation(g, p.act) * u, p.f16);
    }
    __syncthreads();
    if (p.cluster > 1) cluster_sync();  // no CTA leaves while another may still read its shared memory
}

// ---------------------------------------------------------------- elementwise parts

// dg and du, [M, ldp] with ldp a multiple of 8; 8 columns per thread.
__global__ void __launch_bounds__(256) gated_grad_kernel(const uint16_t* g, const uint16_t* u, const uint16_t* dout, uint16_t* dg,
                                                        uint16_t* du, long long M, int F, int ldp, int vec, int f16, int act) {
    const int per_row = ldp / 8;
    const long long n = M * per_row;
    pdl_wait();
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
        const long long m = i / per_row;
        const int c = static_cast<int>(i - m * per_row) * 8;
        const long long o = m * F + c;
        uint16_t a[3][8];
        if (vec) {
            *reinterpret_cast<uint4*>(a[0]) = __ldcs(reinterpret_cast<const uint4*>(g + o));
            *reinterpret_cast<uint4*>(a[1]) = __ldcs(reinterpret_cast<const uint4*>(u + o));
            *reinterpret_cast<uint4*>(a[2]) = __ldcs(reinterpret_cast<const uint4*>(dout + o));
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const bool in = c + e < F;
                a[0][e] = in ? g[o + e] : 0;
                a[1][e] = in ? u[o + e] : 0;
                a[2][e] = in ? dout[o + e] : 0;
            }
        }
        uint32_t wg[4], wu[4];
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            float vg[2], vu[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float av, dv;
                activation_grad(up16(a[0][e + h], f16), act, av, dv);
                const float d = up16(a[2][e + h], f16);
                vg[h] = d * up16(a[1][e + h], f16) * dv;
                vu[h] = d * av;
            }
            wg[e / 2] = pack16(vg[0], vg[1], f16);
            wu[e / 2] = pack16(vu[0], vu[1], f16);
        }
        *reinterpret_cast<uint4*>(dg + m * ldp + c) = make_uint4(wg[0], wg[1], wg[2], wg[3]);
        *reinterpret_cast<uint4*>(du + m * ldp + c) = make_uint4(wu[0], wu[1], wu[2], wu[3]);
    }
    pdl_trigger();
}

// [rows, cols] with any row stride to [rows, ldp] with rows of whole 16-byte vectors.
__global__ void __launch_bounds__(256) pad_rows_kernel(const uint16_t* src, long long ld, uint16_t* dst, long long rows, int cols, int ldp) {
    const int per_row = ldp / 8;
    const long long n = rows * per_row;
    pdl_wait();
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
        const long long r = i / per_row;
        const int c = static_cast<int>(i - r * per_row) * 8;
        uint16_t v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = c + e < cols ? src[r * ld + c + e] : 0;
        *reinterpret_cast<uint4*>(dst + r * ldp + c) = *reinterpret_cast<const uint4*>(v);
    }
    pdl_trigger();
}

// ---------------------------------------------------------------- host side

unsigned stream_grid(long long items) {
    const long long blocks = (items + 255) / 256, cap = static_cast<long long>(sm_count()) * 8;
    return static_cast<unsigned>(blocks < cap ? blocks : cap);
}

// A matrix of rows x cols 16-bit elements.
struct Mat {
    const void* p;
    long long rows, cols, ld;
    bool tma() const { return aligned16(p) && ld % 8 == 0; }
    long long padded() const { return (cols + 7) / 8 * 8; }
    size_t scratch() const { return tma() ? 0 : static_cast<size_t>(rows * padded()) * 2 + 256; }
};

// Pool scratch of one call, handed out in 256-byte steps and returned on the stream.
struct Scratch {
    uint8_t* base = nullptr;
    size_t used = 0;
    cudaStream_t st;
    const char* what;
    int open(size_t bytes) {
        if (bytes == 0) return 0;
        void* mem = nullptr;
        cudaError_t e = pool_malloc(&mem, bytes, st);
        if (e != cudaSuccess) return api_fail(e, "%s: scratch of %zu bytes: %s", what, bytes, cudaGetErrorString(e));
        base = static_cast<uint8_t*>(mem);
        return 0;
    }
    uint16_t* take(size_t bytes) {
        uint16_t* p = reinterpret_cast<uint16_t*>(base + used);
        used += (bytes + 255) / 256 * 256;
        return p;
    }
    int close(int rc) {
        if (!base) return rc;
        cudaError_t e = cudaFreeAsync(base, st);
        return rc == 0 && e != cudaSuccess ? api_fail(e, "%s: %s", what, cudaGetErrorString(e)) : rc;
    }
};

// The matrix as TMA can read it: itself, or its copy in padded scratch.
int ready(Mat& m, Scratch& s, cudaStream_t st) {
    if (m.tma()) return 0;
    const long long ldp = m.padded();
    uint16_t* dst = s.take(static_cast<size_t>(m.rows * ldp) * 2);
    launch_pdl(pad_rows_kernel, stream_grid(m.rows * (ldp / 8)), 256, 0, st, static_cast<const uint16_t*>(m.p), m.ld, dst, m.rows,
               static_cast<int>(m.cols), static_cast<int>(ldp));
    m.p = dst;
    m.ld = ldp;
    return launch_status(s.what);
}

// Map of boxes of box_rows rows by 64 columns.
int map_of(CUtensorMap* t, const Mat& m, uint32_t box_rows, bool f16) {
    return make_map(t, m.p, static_cast<uint64_t>(m.cols), static_cast<uint64_t>(m.rows), 1, static_cast<uint64_t>(m.ld),
                    static_cast<uint64_t>(m.ld) * static_cast<uint64_t>(m.rows), 64, box_rows, f16);
}

template <int MODE, bool A_MN, bool B_MN>
int launch_pair(const Mat& a0, const Mat& a1, const Mat& b0, const Mat& b1, PairParams p, const char* what, cudaStream_t st) {
    using Cfg = PairCfg;
    CUtensorMap ta0, ta1, tb0, tb1;
    const bool f16 = p.f16 != 0;
    // K-major: boxes of 128 rows; MN-major: boxes of 128 K rows
    if (int rc = map_of(&ta0, a0, 128, f16)) return rc;
    if (int rc = map_of(&ta1, a1, 128, f16)) return rc;
    if (int rc = map_of(&tb0, b0, 128, f16)) return rc;
    if (int rc = map_of(&tb1, b1, 128, f16)) return rc;
    CUtensorMap to[3] = {ta0, ta0, ta0};  // of the outputs, where TMA can store them (p.vec)
    for (int i = 0; i < 3; ++i) {
        if (!p.vec || !p.out[i]) continue;
        const Mat o{p.out[i], p.M, p.N, p.ldc};
        if (int rc = map_of(&to[i], o, 32, f16)) return rc;
    }
    const int bn = MODE == FORWARD ? 128 : Cfg::BN;
    p.m_tiles = (p.M + Cfg::BM - 1) / Cfg::BM;
    p.n_tiles = (p.N + bn - 1) / bn;
    const long long tiles = static_cast<long long>(p.m_tiles) * p.n_tiles, total = tiles * (MODE == DW ? 2 : 1);
    if (total > 0x3fffffff) return fail(cudaErrorInvalidValue, "%s: too many output tiles", what);
    p.tiles = static_cast<int>(tiles);
    // The tiles after the last full round of the pairs are cut along K, so that the round they take is as short as
    // the pairs allow: up to 8 cuts of at least 8 K blocks each (the join costs about 5 us).
    const int pairs = sm_count() / 2, rest = static_cast<int>(total % pairs);
    p.cuts = 1;
    while (rest > 0 && p.cuts < 8 && rest * (p.cuts + 1) <= pairs && p.num_kb >= 8 * (p.cuts + 1)) ++p.cuts;
    p.whole = static_cast<int>(total) - (p.cuts > 1 ? rest : 0);
    p.items = p.cuts > 1 ? p.whole + rest * p.cuts : p.whole;
    Scratch parts{nullptr, 0, st, what};
    if (p.cuts > 1) {
        if (int rc = parts.open(static_cast<size_t>(rest * p.cuts) * Cfg::BM * Cfg::BN * sizeof(float))) return rc;
        p.part = reinterpret_cast<float4*>(parts.base);
    }
    auto gated_pair = gated_pair_kernel<MODE, A_MN, B_MN>;
    static SmemLimit limit;
    int rc = limit.ensure(gated_pair, Cfg::SMEM, what);
    if (rc == 0) {
        gated_pair<<<2 * (p.items < pairs ? p.items : pairs), 192, Cfg::SMEM, st>>>(ta0, ta1, tb0, tb1, to[0], to[1], to[2], p);
        rc = launch_status(what);
    }
    if (rc == 0 && p.cuts > 1) {
        const dim3 grid(static_cast<unsigned>(rest), MODE == FORWARD ? 4 : 8);
        launch_pdl(gated_pair_join_kernel<MODE>, grid, 256, 0, st, p);
        rc = launch_status(what);
    }
    return parts.close(rc);
}

// 128 rows: 66.8 us there, 64 as one tile of the pair kernel (4096 -> 14336)
constexpr int kFewRows = 64;

template <int NT, bool W_MN> int launch_rows(const Mat& x, const Mat& g, const Mat& u, RowsParams p, const char* what, cudaStream_t st) {
    constexpr int STAGE = 2 * 128 * 64 * 2 + NT * 64 * 2;
    CUtensorMap tx, tg, tu;
    const bool f16 = p.f16 != 0;
    if (int rc = map_of(&tx, x, NT, f16)) return rc;
    if (int rc = map_of(&tg, g, W_MN ? 64 : 128, f16)) return rc;
    if (int rc = map_of(&tu, u, W_MN ? 64 : 128, f16)) return rc;
    // Deep rings for one CTA per SM, half as deep for two (which also hold the partial sums).
    constexpr int ONE = (220 * 1024) / STAGE < 6 ? (220 * 1024) / STAGE : 6;
    constexpr int TWO = (109 * 1024) / STAGE;
    constexpr int resident = TWO * STAGE >= 2 * NT * 128 * 4 ? 2 : 1;
    // One SM draws about 50 GB/s whatever its ring, so the time is that of the SM with the most work: the cut of
    // K is the one whose busiest SM has the least, the finer one if equal (14336 columns, one row: 41.9 us uncut with
    // one CTA per SM, 39.2 cut in two; 11008 columns, 48 rows: 44.5 us uncut, 43.7 in two, 37.3 in three).
    const int tiles = (p.N + 127) / 128, sms = sm_count();
    p.cluster = 1;
    double least = 0;
    for (int cut = 1; cut <= 8 && (cut == 1 || (tiles * cut <= resident * sms && p.num_kb >= 4 * cut)); ++cut) {
        const int ctas = tiles * cut;
        const double busiest = static_cast<double>((ctas + sms - 1) / sms) / ctas;
        if (cut == 1 || busiest <= least) {
            least = busiest;
            p.cluster = cut;
        }
    }
    p.stages = tiles * p.cluster > sms && resident == 2 ? TWO : ONE;
    const int smem = p.stages * STAGE + 1024;
    auto gated_rows = gated_rows_kernel<NT, W_MN>;
    static SmemLimit limit;
    if (int rc = limit.ensure(gated_rows, smem, what)) return rc;
    if (p.cluster > 1) {
        launch_pdl_cluster(gated_rows, static_cast<unsigned>(tiles * p.cluster), 192, static_cast<unsigned>(p.cluster),
                           static_cast<size_t>(smem), st, tx, tg, tu, p);
    } else {
        launch_pdl(gated_rows, static_cast<unsigned>(tiles), 192, static_cast<size_t>(smem), st, tx, tg, tu, p);
    }
    return launch_status(what);
}

template <bool W_MN> int forward_rows(const Mat& x, const Mat& g, const Mat& u, const RowsParams& p, const char* what, cudaStream_t st) {
    if (p.M <= 16) return launch_rows<16, W_MN>(x, g, u, p, what, st);
    if (p.M <= 32) return launch_rows<32, W_MN>(x, g, u, p, what, st);
    return launch_rows<64, W_MN>(x, g, u, p, what, st);
}

int check(const char* what, int dt, int act, size_t M, size_t D, size_t F, size_t ldx, size_t ldw, bool trans) {
    const size_t most = size_t{1} << 30;
    if (dt != DT_BF16 && dt != DT_F16) return fail(cudaErrorInvalidValue, "%s: unsupported dtype %d", what, dt);
    if (act < ACT_SILU || act > ACT_GELU_TANH) return fail(cudaErrorInvalidValue, "%s: unknown activation %d", what, act);
    if (D == 0 || F == 0 || D > most || F > most || M > most) return fail(cudaErrorInvalidValue, "%s: extents %zu, %zu, %zu", what, M, D, F);
    if (ldx < D || ldx > (size_t{1} << 35)) return fail(cudaErrorInvalidValue, "%s: row stride %zu of x below %zu", what, ldx, D);
    const size_t wcols = trans ? D : F;
    if (ldw < wcols || ldw > (size_t{1} << 35)) return fail(cudaErrorInvalidValue, "%s: row stride %zu of the weights below %zu", what, ldw, wcols);
    return 0;
}

// Whether the output o, if there is one, is any of the tensors given.
template <typename... P> bool is_any(const void* o, const P*... p) { return o && ((static_cast<const void*>(p) == o) || ...); }

template <typename... P> bool aligned2(const P*... p) { return (((reinterpret_cast<uintptr_t>(p)) | ...) & 1u) == 0; }

}  // namespace

int gated_linear_status_take(int* code) {
    int zero = 0;
    cudaError_t e = cudaMemcpyFromSymbol(code, g_gated_status, sizeof(int));
    if (e == cudaSuccess) e = cudaMemcpyToSymbol(g_gated_status, &zero, sizeof(int));
    return static_cast<int>(e);
}

}  // namespace bee_b200

using namespace bee_b200;

extern "C" {

int bee_b200_gated_linear(int dt, int act, const void* x, size_t ldx, const void* wg, const void* wu, size_t ldw, int trans,
                          void* out, void* g, void* u, size_t M, size_t D, size_t F, bee_b200_stream_t stream) {
    const char* what = "gated_linear";
    if (int rc = check(what, dt, act, M, D, F, ldx, ldw, trans != 0)) return rc;
    if (M == 0) return ok();
    if (!x || !wg || !wu || !out || !g != !u) return fail(cudaErrorInvalidValue, "%s: null pointer", what);
    if (!aligned2(x, wg, wu, out, g, u)) return fail(cudaErrorInvalidValue, "%s: a tensor is not aligned to its type", what);
    if (is_any(out, x, wg, wu, g, u) || is_any(g, x, wg, wu, u) || is_any(u, x, wg, wu))
        return fail(cudaErrorInvalidValue, "%s: outputs must not overlap the inputs or each other", what);
    cudaStream_t st = as_stream(stream);
    const long long m = static_cast<long long>(M), d = static_cast<long long>(D), f = static_cast<long long>(F);
    const long long lw = static_cast<long long>(ldw);
    Mat mx{x, m, d, static_cast<long long>(ldx)};
    Mat mg{wg, trans ? f : d, trans ? d : f, lw}, mu{wu, trans ? f : d, trans ? d : f, lw};
    Scratch s{nullptr, 0, st, what};
    if (int rc = s.open(mx.scratch() + mg.scratch() + mu.scratch())) return rc;
    int rc = ready(mx, s, st);
    if (rc == 0) rc = ready(mg, s, st);
    if (rc == 0) rc = ready(mu, s, st);
    if (rc == 0 && m <= kFewRows) {
        RowsParams p{};
        p.M = static_cast<int>(m);
        p.N = static_cast<int>(f);
        p.num_kb = static_cast<int>((d + 63) / 64);
        p.out[0] = static_cast<uint16_t*>(out);
        p.out[1] = static_cast<uint16_t*>(g);
        p.out[2] = static_cast<uint16_t*>(u);
        p.f16 = dt == DT_F16;
        p.act = act;
        rc = trans ? forward_rows<false>(mx, mg, mu, p, what, st) : forward_rows<true>(mx, mg, mu, p, what, st);
    } else if (rc == 0) {
        PairParams p{};
        p.M = static_cast<int>(m);
        p.N = static_cast<int>(f);
        p.num_kb = static_cast<int>((d + PairCfg::BK - 1) / PairCfg::BK);
        p.ldc = f;
        p.out[0] = static_cast<uint16_t*>(out);
        p.out[1] = static_cast<uint16_t*>(g);
        p.out[2] = static_cast<uint16_t*>(u);
        p.vec = f % 8 == 0 && aligned16(out) && aligned16(g) && aligned16(u);
        p.f16 = dt == DT_F16;
        p.act = act;
        rc = trans ? launch_pair<FORWARD, false, false>(mx, mx, mg, mu, p, what, st) : launch_pair<FORWARD, false, true>(mx, mx, mg, mu, p, what, st);
    }
    return s.close(rc);
}

int bee_b200_gated_linear_backward(int dt, int act, const void* x, size_t ldx, const void* wg, const void* wu, size_t ldw,
                                   int trans, const void* g, const void* u, const void* dout, void* dx, void* dwg, void* dwu,
                                   size_t lddw, size_t M, size_t D, size_t F, bee_b200_stream_t stream) {
    const char* what = "gated_linear_backward";
    if (int rc = check(what, dt, act, M, D, F, ldx, ldw, trans != 0)) return rc;
    if (!dwg != !dwu || (!dx && !dwg)) return fail(cudaErrorInvalidValue, "%s: null pointer", what);
    const size_t wrows = trans ? F : D, wcols = trans ? D : F;
    if (dwg && (lddw < wcols || lddw > (size_t{1} << 35)))
        return fail(cudaErrorInvalidValue, "%s: row stride %zu of the weights' gradients below %zu", what, lddw, wcols);
    cudaStream_t st = as_stream(stream);
    if (M == 0) {  // sums over no rows
        if (!dwg) return ok();
        cudaError_t e = cudaMemset2DAsync(dwg, lddw * 2, 0, wcols * 2, wrows, st);
        if (e == cudaSuccess) e = cudaMemset2DAsync(dwu, lddw * 2, 0, wcols * 2, wrows, st);
        return e == cudaSuccess ? ok() : api_fail(e, "%s: %s", what, cudaGetErrorString(e));
    }
    if (!g || !u || !dout || (dx && (!wg || !wu)) || (dwg && !x)) return fail(cudaErrorInvalidValue, "%s: null pointer", what);
    if (!aligned2(x, wg, wu, g, u, dout, dx, dwg, dwu)) return fail(cudaErrorInvalidValue, "%s: a tensor is not aligned to its type", what);
    if (is_any(dx, x, wg, wu, dwg, dwu) || is_any(dwg, x, wg, wu, dwu) || is_any(dwu, x, wg, wu))
        return fail(cudaErrorInvalidValue, "%s: gradients must not overlap the inputs or each other", what);
    const long long m = static_cast<long long>(M), d = static_cast<long long>(D), f = static_cast<long long>(F);
    const long long lw = static_cast<long long>(ldw);
    Mat mx{x, m, d, static_cast<long long>(ldx)};
    Mat mg{wg, trans ? f : d, trans ? d : f, lw}, mu{wu, trans ? f : d, trans ? d : f, lw};
    Mat dg{nullptr, m, f, (f + 7) / 8 * 8}, du = dg;
    const size_t grad_bytes = static_cast<size_t>(m * dg.ld) * 2;
    Scratch s{nullptr, 0, st, what};
    if (int rc = s.open(2 * (grad_bytes + 256) + (dwg ? mx.scratch() : 0) + (dx ? mg.scratch() + mu.scratch() : 0))) return rc;
    uint16_t *pdg = s.take(grad_bytes), *pdu = s.take(grad_bytes);
    dg.p = pdg;
    du.p = pdu;
    const int f16 = dt == DT_F16;
    const int vec = f % 8 == 0 && aligned16(g) && aligned16(u) && aligned16(dout);
    launch_pdl(gated_grad_kernel, stream_grid(m * (dg.ld / 8)), 256, 0, st, static_cast<const uint16_t*>(g), static_cast<const uint16_t*>(u),
               static_cast<const uint16_t*>(dout), pdg, pdu, m, static_cast<int>(f), static_cast<int>(dg.ld), vec, f16, act);
    int rc = launch_status(what);
    if (rc == 0 && dx) {
        rc = ready(mg, s, st);
        if (rc == 0) rc = ready(mu, s, st);
        PairParams p{};
        p.M = static_cast<int>(m);
        p.N = static_cast<int>(d);
        p.half_kb = static_cast<int>((f + PairCfg::BK - 1) / PairCfg::BK);
        p.num_kb = 2 * p.half_kb;
        p.ldc = d;
        p.out[0] = static_cast<uint16_t*>(dx);
        p.vec = d % 8 == 0 && aligned16(dx);
        p.f16 = f16;
        // weights [F, D] have the output's columns contiguous, [D, F] the contraction's
        if (rc == 0) rc = trans ? launch_pair<DX, false, true>(dg, du, mg, mu, p, what, st) : launch_pair<DX, false, false>(dg, du, mg, mu, p, what, st);
    }
    if (rc == 0 && dwg) {
        rc = ready(mx, s, st);
        PairParams p{};
        p.M = static_cast<int>(wrows);
        p.N = static_cast<int>(wcols);
        p.num_kb = static_cast<int>((m + PairCfg::BK - 1) / PairCfg::BK);
        p.ldc = static_cast<long long>(lddw);
        p.out[0] = static_cast<uint16_t*>(dwg);
        p.out[1] = static_cast<uint16_t*>(dwu);
        p.vec = lddw % 8 == 0 && wcols % 8 == 0 && aligned16(dwg) && aligned16(dwu);  // else what follows a row would be written
        p.f16 = f16;
        p.a_second = trans ? 1 : 0;
        if (rc == 0) rc = trans ? launch_pair<DW, true, true>(dg, du, mx, mx, p, what, st) : launch_pair<DW, true, true>(mx, mx, dg, du, p, what, st);
    }
    return s.close(rc);
}

}  // extern "C"
