// Matrix products grouped by expert: slot s of a row list sorted by expert multiplies the weights of its expert,
//
//   y[s, :] = act(x[rows[s], :] . w[e]^T + bias[e]),   offsets[e] <= s < offsets[e + 1],
//   gated:  y[s, n] = act(v[n]) * v[N + n],  v = x . w[e]^T + bias[e] over the expert's 2N weight rows.
//
// The groups are ragged and known on the device only.  A wave cuts them into tiles with one scan over the offsets in
// registers; the workgroups, at most as many as the GPU holds at once, walk the tiles in that order.  Slots behind
// offsets[experts] are zeros.
//
// Weights are [N, K] and rows [*, K], both with K contiguous, so both operands of a 16 x 16 matrix instruction are 16-byte
// pieces along K: lane l holds row l & 15, piece l >> 4.  The weights are the first operand: a lane's four results are
// then four consecutive columns of one row of y.  float32 takes four 16x16x4 instructions over the same 16 bytes (the
// k of a lane's j-th float is the same for both operands, which is all the sum needs).  Sums are held in float32.
#include "fd_conv_split_dev.h"
#include "fd_elem.h"

#include <atomic>
#include <cmath>
#include <type_traits>

namespace fd {

struct ExpertArgs {
    const void *x, *w, *bias;
    void* y;
    const int32_t *offsets, *rows;
    int64_t x_rows;
    int K, N, wrows, experts, slots, act, gated, tiles_n;
};

template <typename T>
__device__ __forceinline__ f32x4_t mma(u32x4_t a, u32x4_t b, f32x4_t c);
template <>
__device__ __forceinline__ f32x4_t mma<_Float16>(u32x4_t a, u32x4_t b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x4_t mma<__bf16>(u32x4_t a, u32x4_t b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

template <typename T>
__device__ __forceinline__ f32x4_t mma_piece(u32x4_t w, u32x4_t x, f32x4_t c) {
    if constexpr (sizeof(T) == 2) return mma<T>(w, x, c);
    const f32x4_t fw = __builtin_bit_cast(f32x4_t, w), fx = __builtin_bit_cast(f32x4_t, x);
#pragma unroll
    for (int t = 0; t < 4; ++t) c = __builtin_amdgcn_mfma_f32_16x16x4f32(fw[t], fx[t], c, 0, 0, 0);
    return c;
}

// all NI x MI tiles of one 16-byte piece; in float32 the four instructions of a tile are kept apart
template <typename T, int NI, int MI>
__device__ __forceinline__ void mma_block(const u32x4_t (&w)[NI], const u32x4_t (&x)[MI], f32x4_t (&acc)[NI][MI]) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int j = 0; j < MI; ++j) acc[i][j] = mma<T>(w[i], x[j], acc[i][j]);
    } else {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int j = 0; j < MI; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(f32x4_t, w[i])[t], __builtin_bit_cast(f32x4_t, x[j])[t],
                                                                     acc[i][j], 0, 0, 0);
    }
}

// one row fragment's tiles of it
template <typename T, int NI, int MI>
__device__ __forceinline__ void mma_column(const u32x4_t (&w)[NI], const u32x4_t& x, f32x4_t (&acc)[NI][MI], int j) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < NI; ++i) acc[i][j] = mma<T>(w[i], x, acc[i][j]);
    } else {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < NI; ++i)
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(f32x4_t, w[i])[t], __builtin_bit_cast(f32x4_t, x)[t],
                                                                 acc[i][j], 0, 0, 0);
    }
}

// 16 bytes of a row, elements from `left` on as zeros
template <typename T>
__device__ __forceinline__ u32x4_t load_piece(const T* p, int left) {
    constexpr int V = 16 / (int)sizeof(T);
    T raw[V];
    if (left >= V) {
        __builtin_memcpy(raw, p, 16);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) raw[i] = i < left ? p[i] : (T)0.f;
    }
    u32x4_t v;
    __builtin_memcpy(&v, raw, 16);
    return v;
}

// v * Phi(v).  Phi(v) = erfc(z) / 2 for v < 0 and 1 - erfc(z) / 2 otherwise, z = |v| / sqrt(2).
// 16-bit results: erfc(z) / 2 = exp(-z^2) * (c1 t + .. + c7 t^7), t = 1 / (1 + 0.515 z), whose polynomial is fitted to
// exp(z^2) erfc(z) / 2 over 0 <= z <= 10.5 for the least RELATIVE error, 8.5e-7, by linear programming.  The result is then good in
// the negative tail too, where it is as small as exp(-z^2): the fit, seven terms and the argument of exp2 are off by less than (48 + 1.5 v^2) * 2^-24
// of the value, a fortieth of half a step of float16 down to its smallest numbers (v = -5.6) and less of bfloat16 (v = -13).
template <typename T>
__device__ __forceinline__ float gelu(float v) {
    if (sizeof(T) == 4) return 0.5f * v * erfcf(-0.70710678118654752f * v);     // no cancellation for v << 0
    const float t = __builtin_amdgcn_rcpf(1.f + 0.36415999f * fabsf(v));       // 0.515 / sqrt(2)
    const float half = t * (0.145349710f + t * (0.143801985f + t * (0.138411605f + t * (0.033301960f +
                       t * (0.168811180f + t * (-0.177848335f + t * 0.048172315f))))));
    const float tail = half * __builtin_amdgcn_exp2f(-0.72134752044448170f * v * v);              // erfc(z) / 2
    return v * (v < 0.f ? tail : 1.f - tail);
}

template <typename T>
__device__ __forceinline__ float activate(float v, int act) {
    if (act == FD_ACT_RELU) return v < 0.f ? 0.f : v;         // not a number stays so
    // 16-bit results: the hardware's exp2 and reciprocal, off by less than (1.5 |v| + 8) * 2^-24 of the value, a hundredth of half a
    // step; zero from v = -87.3 on, where the value is below 100 * 2^-126 (the form for float32: 1133 against 1110 us for the
    // gated product of 261120 slots, 64 experts, 1024 -> 2 x 1024 in bfloat16)
    if (act == FD_ACT_SILU && sizeof(T) == 2) return v * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504088896341f * v));
    if (act == FD_ACT_SILU) {
        // v * e / (1 + e) for v < 0 and v / (1 + e) otherwise, e = exp(-|v|): nothing overflows, at most 12 * 2^-24 of the value (a
        // quotient in place of the hardware's reciprocal cost 4 % of a product of 1024 inputs)
        const float e = exp_fast(-fabsf(v));
        return (v < 0.f ? v * e : v) * __builtin_amdgcn_rcpf(1.f + e);
    }
    if (act == FD_ACT_GELU) return gelu<T>(v);
    return v;
}

// The same value, of which the compiler knows nothing: what is computed from it stays where it stands.  Addresses that are
// needed once a tile would otherwise be computed before the loop over tiles and held, or spilled, through all of it.
__device__ __forceinline__ int opaque(int v) {
    asm volatile("" : "+v"(v));
    return v;
}

// Between what a wave's lanes write to LDS and what other lanes of it read there: the accesses of a wave are carried out in their
// order, which the compiler keeps only between those of one lane.
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// The tiles of all groups when every group is cut into tiles of BM slots, one scan over the offsets by every wave: lane l
// takes the same number of consecutive groups as any other, they start at slot `start` and have `tiles` tiles from
// `first` on.  Ends are clamped to [0, slots] and never decrease, so any content of `offsets` stays in bounds.  `ends`
// (LDS, one word a group) keeps what a lane read of its groups; all waves write the same.
struct TileScan {
    int start, first, tiles, total, routed;      // routed: the slots that belong to an expert
};

__device__ __forceinline__ TileScan scan_tiles(const ExpertArgs& a, int bm, int* ends) {
    const int lane = threadIdx.x & 63, per = (a.experts + 63) / 64;
    int upto = 0;
    for (int i = lane * per; i < min((lane + 1) * per, a.experts); ++i) {
        upto = max(upto, min(a.offsets[i + 1], a.slots));
        ends[i] = upto;
    }
    const int most = wave_scan<true>(upto);
    TileScan t;
    t.routed = __builtin_amdgcn_readlane(most, 63);
    t.start = __builtin_amdgcn_update_dpp(0, most, 0x138, 0xf, 0xf, false);       // the lane before's; 0 in the first
    t.tiles = 0;
    int at = t.start;
    for (int i = lane * per; i < min((lane + 1) * per, a.experts); ++i) {
        const int to = max(at, ends[i]);
        t.tiles += (to - at + bm - 1) / bm;
        at = to;
    }
    const int sum = wave_scan<false>(t.tiles);
    t.first = sum - t.tiles;
    t.total = __builtin_amdgcn_readlane(sum, 63);
    return t;
}

// Tile `tile` (below the total): slots [m0, m1) of expert e.
__device__ __forceinline__ void locate_tile(const TileScan& t, const ExpertArgs& a, const int* ends, int bm, int tile, int& e, int& m0, int& m1) {
    const int lane = opaque(threadIdx.x & 63), per = (a.experts + 63) / 64;
    const bool mine = tile >= t.first && tile < t.first + t.tiles;
    int fe = 0, f0 = 0, f1 = 0;
    if (mine) {
        int at = t.start, first = t.first;
        for (int i = lane * per; i < min((lane + 1) * per, a.experts); ++i) {
            const int to = max(at, ends[i]);
            const int n = (to - at + bm - 1) / bm;
            if (tile >= first && tile < first + n) {
                fe = i;
                f0 = at + (tile - first) * bm;
                f1 = min(to, f0 + bm);
            }
            first += n;
            at = to;
        }
    }
    const int src = __ffsll((unsigned long long)__ballot(mine)) - 1;
    e = __builtin_amdgcn_readlane(fe, src);
    m0 = __builtin_amdgcn_readlane(f0, src);
    m1 = __builtin_amdgcn_readlane(f1, src);
}

// The tiles of this workgroup: workgroup i runs on XCD i mod 8, and each XCD walks a contiguous eighth of the tiles (columns
// fastest), so that the tiles that share rows and weights share an L2.  The grid is a multiple of 8.
struct TileWalk {
    int next, end, by;
};

__device__ __forceinline__ TileWalk walk_tiles(const TileScan& t, const ExpertArgs& a) {
    const int n = t.total * a.tiles_n, q = n >> 3, r = n & 7, xcd = blockIdx.x & 7;
    TileWalk w;
    const int begin = xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q;
    w.end = begin + q + (xcd < r ? 1 : 0);
    w.next = begin + (blockIdx.x >> 3);
    w.by = gridDim.x >> 3;
    return w;
}

// The slots that belong to nobody, the last ones of y, by all workgroups together.
template <typename T>
__device__ __forceinline__ void zero_rest(const ExpertArgs& a, int routed) {
    const int64_t n = (int64_t)(a.slots - routed) * a.N;
    T* p = (T*)a.y + (int64_t)routed * a.N;
    const float zero[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int64_t i = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) * 8; i < n; i += (int64_t)gridDim.x * blockDim.x * 8)
        store8(p + i, (int)min<int64_t>(n - i, 8), zero);
}

// The row of x that slot s multiplies, -1 for none (a negative or too large index reads as a row of zeros).
__device__ __forceinline__ int64_t source_row(const ExpertArgs& a, int s) {
    const int64_t r = a.rows ? a.rows[s] : s;
    return r >= 0 && r < a.x_rows ? r : -1;
}

// Weight row of row r of a tile that starts at output column n0 (-1: none).  Gated tiles alternate 16 rows of the
// first half with the 16 rows of the second half that multiply them, so both land in the same lane.
__device__ __forceinline__ int weight_row(const ExpertArgs& a, int n0, int r) {
    if (!a.gated) return n0 + r < a.N ? n0 + r : -1;
    const int n = n0 + (r >> 5) * 16 + (r & 15);
    return n < a.N ? ((r >> 4) & 1) * a.N + n : -1;
}

// Results of a wave (rows from m0 on, weight rows wn .. of the tile that starts at output column n0) through `part`, the wave's
// own piece of LDS: the float32 sums go in as they lie in registers, come back as 8 consecutive columns of a row, and
// bias, activation, gate and the one rounding happen on the way to a full-width store.  The 16-byte piece c of row r lies
// at c ^ (r & 15), without which the 16 rows of a write would share their banks.
template <typename T, int NI, int MI, int BYTES>
__device__ __forceinline__ void store_tile(const ExpertArgs& a, int e, int m0, int m1, int n0, int wn, const f32x4_t (&acc)[NI][MI], char* part) {
    constexpr int ROW = NI * 64;                                       // bytes of a row of NI * 16 sums
    constexpr int FIT = BYTES / (16 * ROW), JP = FIT >= MI ? MI : (FIT >= 4 ? 4 : (FIT >= 2 ? 2 : 1));
    constexpr int MASK = NI * 4 - 1 < 15 ? NI * 4 - 1 : 15;
    static_assert(JP >= 1 && JP * 16 * ROW <= BYTES && MI % JP == 0 && (NI & (NI - 1)) == 0, "a wave's piece of LDS holds 16 rows");
    const int lane = opaque(threadIdx.x & 63);
    // pieces of 8 output columns in a row; a lane stays with one of them and takes every (64 / pieces)-th row
    const int pieces = a.gated ? NI : 2 * NI, q = lane & (pieces - 1), shift = __builtin_ctz(pieces);
    const int n = n0 + (a.gated ? wn / 2 : wn) + q * 8, left = a.N - n;
    const int c = a.gated ? (q >> 1) * 8 + (q & 1) * 2 : q * 2;                  // gated: 16 columns of the first half, 16 of the second
    float b1[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, b2[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (a.bias) {
        const T* bias = (const T*)a.bias + (int64_t)e * a.wrows + n;
        load8(bias, left, b1);
        if (a.gated) load8(bias + a.N, left, b2);
    }
#pragma unroll
    for (int p = 0; p < MI / JP; ++p) {
#pragma unroll
        for (int j = 0; j < JP; ++j)
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int r = j * 16 + (lane & 15), at = i * 4 + (lane >> 4);
                *(f32x4_t*)(part + r * ROW + ((at ^ (r & MASK)) * 16)) = acc[i][p * JP + j];
            }
        wave_fence();
        for (int r = lane >> shift; r < JP * 16; r += 64 >> shift) {
            const int m = m0 + p * JP * 16 + r;
            if (m >= m1 || left <= 0) break;
            auto read = [&](int at, float* to) {
                const f32x4_t lo = *(const f32x4_t*)(part + r * ROW + ((at ^ (r & MASK)) * 16));
                const f32x4_t hi = *(const f32x4_t*)(part + r * ROW + (((at + 1) ^ (r & MASK)) * 16));
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    to[i] = lo[i];
                    to[4 + i] = hi[i];
                }
            };
            float v[8];
            read(c, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] += b1[i];
            if (a.act) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = activate<T>(v[i], a.act);
            }
            if (a.gated) {
                float u[8];
                read(c + 4, u);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] *= u[i] + b2[i];
            }
            store8((T*)a.y + (int64_t)m * a.N + n, left, v);
        }
        wave_fence();
    }
}

// ---------------------------------------------------------------------------------------------------------------
// Tile kernel for rows of any length and alignment: BM slots x BN weight rows, 4 waves of (BM/2) x (BN/2), 128 bytes of K a
// step, operands through registers (D steps ahead) into two LDS stages.  Loads that are not aligned are what bounds it (2331
// slots, 333 x 1001 float16: 16.5 us with 64 x 64 tiles, 14.4 with 32 x 64, of which 8.2 and 6.5 are the launch, the scan, the row
// list, the store and the first two steps; 333 x 1024: 10.8 with both).
// Reading the aligned pieces that cover a row and shifting them on the way to LDS took 17.7, more steps ahead no less.
// A row of a step is 8 pieces; piece c of row r lies at c ^ ((r >> 1) & 7), which spreads the fragment reads over the banks.
template <typename T, int BM, int BN, int D, int OCC>
__global__ __launch_bounds__(256, OCC) void expert_tile_kernel(ExpertArgs a) {
    constexpr int V = 16 / (int)sizeof(T), BK = 8 * V, ROWS = BM + BN;
    constexpr int RA = BM / 32, RB = BN / 32, MI = BM / 32, NI = BN / 32;
    __shared__ u32x4_t smem[2][ROWS * 8];
    __shared__ int ends[FD_EXPERT_MAX];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const TileScan scan = scan_tiles(a, BM, ends);
    zero_rest<T>(a, scan.routed);
    const TileWalk walk = walk_tiles(scan, a);
    const int c = tid & 7, r0 = tid >> 3, pos = c ^ ((r0 >> 1) & 7);
    const int wm = (wave >> 1) * (BM / 2), wn = (wave & 1) * (BN / 2);
    const int steps = (a.K + BK - 1) / BK;
    for (int tile = walk.next; tile < walk.end; tile += walk.by) {
        int e, m0, m1;
        locate_tile(scan, a, ends, BM, tile / a.tiles_n, e, m0, m1);
        const int n0 = (tile % a.tiles_n) * (a.gated ? BN / 2 : BN);
        // Rows that a tile does not have read as some row that exists, their results are not stored; a row that the list
        // does not name reads as zeros.
        const T *xp[RA], *wp[RB];
        bool none[RA];
#pragma unroll
        for (int i = 0; i < RA; ++i) {
            const int64_t r = source_row(a, min(m0 + r0 + 32 * i, m1 - 1));
            none[i] = r < 0;
            xp[i] = a.x_rows ? (const T*)a.x + (r < 0 ? 0 : r) * a.K : (const T*)a.w;
        }
#pragma unroll
        for (int i = 0; i < RB; ++i) {
            const int r = weight_row(a, n0, r0 + 32 * i);
            wp[i] = (const T*)a.w + ((int64_t)e * a.wrows + (r < 0 ? 0 : r)) * a.K;
        }
        f32x4_t acc[NI][MI];
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int j = 0; j < MI; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};

        u32x4_t xr[D][RA], wr[D][RB];
        auto fetch = [&](int step, u32x4_t (&x)[RA], u32x4_t (&w)[RB]) {
            const int at = step * BK + c * V;
            if ((step + 1) * BK <= a.K) {
#pragma unroll
                for (int i = 0; i < RA; ++i) __builtin_memcpy(&x[i], xp[i] + at, 16);
#pragma unroll
                for (int i = 0; i < RB; ++i) __builtin_memcpy(&w[i], wp[i] + at, 16);
            } else {
#pragma unroll
                for (int i = 0; i < RA; ++i) x[i] = load_piece(xp[i] + at, a.K - at);
#pragma unroll
                for (int i = 0; i < RB; ++i) w[i] = load_piece(wp[i] + at, a.K - at);
            }
        };
#pragma unroll
        for (int d = 0; d < D; ++d)
            if (d < steps) fetch(d, xr[d], wr[d]);
        for (int first = 0; first < steps; first += D) {
#pragma unroll
            for (int d = 0; d < D; ++d) {
                const int step = first + d;
                if (step >= steps) break;
                u32x4_t* stage = smem[step & 1];
#pragma unroll
                for (int i = 0; i < RA; ++i) stage[(r0 + 32 * i) * 8 + pos] = none[i] ? u32x4_t{0, 0, 0, 0} : xr[d][i];
#pragma unroll
                for (int i = 0; i < RB; ++i) stage[(BM + r0 + 32 * i) * 8 + pos] = wr[d][i];
                if (step + D < steps) fetch(step + D, xr[d], wr[d]);
                pipeline_barrier();
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    u32x4_t xf[MI], wf[NI];
                    const int at = (h * 4 + (lane >> 4)) ^ ((lane >> 1) & 7);
#pragma unroll
                    for (int i = 0; i < NI; ++i) wf[i] = stage[(BM + wn + i * 16 + (lane & 15)) * 8 + at];
#pragma unroll
                    for (int j = 0; j < MI; ++j) xf[j] = stage[(wm + j * 16 + (lane & 15)) * 8 + at];
                    mma_block<T>(wf, xf, acc);
                }
            }
        }
        __syncthreads();
        store_tile<T, NI, MI, ROWS * 64>(a, e, m0 + wm, m1, n0, wn, acc, (char*)smem + wave * ROWS * 64);
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------------------------------------------
// The same tile with both operands loaded straight into LDS (`buffer_load_dwordx4 ... lds`): no staging registers, and
// rows that do not exist and pieces behind K are zeros by the buffer's range check.  Needs 16-byte aligned rows and
// 31-bit offsets, and two steps or more.  WM x WN waves, two LDS stages, one barrier a step.
template <typename T, int BM, int BN, int WM, int WN, int OCC>
__global__ __launch_bounds__(WM * WN * 64, OCC) void expert_dma_kernel(ExpertArgs a, unsigned x_bytes) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int WAVES = WM * WN, GA = BM / 8 / WAVES, GB = BN / 8 / WAVES, STAGE = (BM + BN) * 128;
    constexpr int MI = BM / WM / 16, NI = BN / WN / 16, EARLY = 0;
    constexpr unsigned NONE = 0x80000000u;
    static_assert(GA * WAVES * 8 == BM && GB * WAVES * 8 == BN, "whole 8-row loads a wave");
    // one array: the compiler waits for all loads into LDS before it reads an array of its own
    __shared__ __attribute__((aligned(16))) char smem[2 * STAGE + (FD_EXPERT_MAX + BM) * 4];
    int *ends = (int*)(smem + 2 * STAGE), *list = ends + FD_EXPERT_MAX;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const TileScan scan = scan_tiles(a, BM, ends);
    zero_rest<T>(a, scan.routed);
    TileWalk walk = walk_tiles(scan, a);
    if (walk.next >= walk.end) return;
    const int row_bytes = a.K * (int)sizeof(T), pieces = row_bytes / 16, steps = (pieces + 7) / 8;
    // Lane l loads 16 bytes of row l / 8 of every 8-row load, the piece that goes to position l % 8.  (r >> 1) & 7 is
    // the same for all loads of a lane: they lie 8 * WAVES rows apart, and WAVES is even.
    const int lrow = wave * 8 + (lane >> 3), piece = (lane & 7) ^ ((lrow >> 1) & 7);

    struct Tile {
        int e, m0, m1, n0;
    };
    // which tile, and a request for its part of the row list, which goes to LDS like the rows
    auto locate = [&](int tile) {
        Tile t;
        locate_tile(scan, a, ends, BM, tile / a.tiles_n, t.e, t.m0, t.m1);
        t.n0 = (tile % a.tiles_n) * (a.gated ? BN / 2 : BN);
        if (a.rows && wave < BM / 64) {
            const __amdgpu_buffer_rsrc_t lr = __builtin_amdgcn_make_buffer_rsrc((void*)(a.rows + t.m0), 0, (unsigned)(t.m1 - t.m0) * 4, 0x00020000);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(lr, (__attribute__((address_space(3))) void*)(list + wave * 64), 4,
                                                     (wave * 64 + lane) * 4, 0, 0, 0);
        }
        return t;
    };
    unsigned xo[GA], wo[GB];                      // byte offset of the lane's piece of step 0, NONE for no row
    auto address = [&](const Tile& t) {
        const int64_t limit = a.rows ? a.x_rows : BM;
#pragma unroll
        for (int i = 0; i < GA; ++i) {
            const int r = lrow + WAVES * 8 * i, src = a.rows ? list[r] : r;
            xo[i] = src >= 0 && src < limit && t.m0 + r < t.m1 ? (unsigned)src * row_bytes + piece * 16 : NONE;
        }
#pragma unroll
        for (int i = 0; i < GB; ++i) {
            const int src = weight_row(a, t.n0, lrow + WAVES * 8 * i);
            wo[i] = src < 0 || t.m0 >= t.m1 ? NONE : (unsigned)src * row_bytes + piece * 16;
        }
    };
    // what is loaded: a tile's rows and weights, their buffers, and whether the lane's piece of the step lies behind K
    __amdgpu_buffer_rsrc_t xr, wr;
    auto aim = [&](const Tile& t) {
        // without a row list the rows of a tile are a range of their own, so x may be of any size; a row at least, so that the
        // offset of a step never passes the end, which the range check subtracts it from
        xr = __builtin_amdgcn_make_buffer_rsrc((void*)((const char*)a.x + (a.rows ? 0 : (int64_t)t.m0 * row_bytes)), 0,
                                               a.rows ? x_bytes : (unsigned)max(t.m1 - t.m0, 1) * row_bytes, 0x00020000);
        wr = __builtin_amdgcn_make_buffer_rsrc((void*)((const char*)a.w + (int64_t)t.e * a.wrows * row_bytes), 0, (unsigned)a.wrows * row_bytes,
                                               0x00020000);
    };
    auto load = [&](int i, int step, int stage) {
        char* base = smem + stage * STAGE + wave * 1024;
        const bool none = step * 8 + piece >= pieces;
        if (i < GA)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(xr, (__attribute__((address_space(3))) void*)(base + WAVES * i * 1024), 16,
                                                     none ? NONE : xo[i < GA ? i : 0], step * 128, 0, 0);
        else
            __builtin_amdgcn_raw_ptr_buffer_load_lds(wr, (__attribute__((address_space(3))) void*)(base + BM * 128 + WAVES * (i - GA) * 1024), 16,
                                                     none ? NONE : wo[i >= GA ? i - GA : 0], step * 128, 0, 0);
    };
    auto issue = [&](int step, int stage) {
#pragma unroll
        for (int i = 0; i < GA + GB; ++i) load(i, step, stage);
    };
    const int wm = (wave / WN) * (BM / WM), wn = (wave % WN) * (BN / WN);
    const int frow = lane & 15, sw = (frow >> 1) & 7;
    int xf_off[2], wf_off[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int pos = ((h * 4 + (lane >> 4)) ^ sw) * 16;
        xf_off[h] = (wm + frow) * 128 + pos;
        wf_off[h] = (BM + wn + frow) * 128 + pos;
    }

    // One pipeline over all steps of all tiles.  Fragments are read half a step ahead: a row fragment is replaced by that
    // of the next half as soon as its products are issued, the weight fragments have two sets.  Early in the second
    // half, when all of the stage has been read, the next step's data is awaited and the stage goes to the load of the step
    // after next.  The last step of a tile leaves its stage to the results; the next tile's first step lies in the
    // other one already.
    u32x4_t xf[MI], wf[2][NI];
    auto read_x = [&](int stage, int h, int j) { xf[j] = *(const u32x4_t*)(smem + stage * STAGE + xf_off[h] + j * 2048); };
    auto read_w = [&](int stage, int h) {
#pragma unroll
        for (int i = 0; i < NI; ++i) wf[h][i] = *(const u32x4_t*)(smem + stage * STAGE + wf_off[h] + i * 2048);
    };
    Tile cur = locate(walk.next);
    wait_vmcnt<0>();
    pipeline_barrier();
    address(cur);
    aim(cur);
    issue(0, 0);
    wait_vmcnt<0>();
    pipeline_barrier();
    read_w(0, 0);
#pragma unroll
    for (int j = 0; j < MI; ++j) read_x(0, 0, j);
    int stage = 0;
    // One step.  KIND 0 loads the current tile's step after next, KIND 1 (the last but one) the next tile's first, KIND 2 (the
    // last) nothing: its stage is left to the results.  The loads go out between the products.
    auto run = [&](auto kind, int step, const Tile& nxt, f32x4_t (&acc)[NI][MI]) {
        constexpr int KIND = decltype(kind)::value, SLOTS = MI - 1 - EARLY, N = GA + GB;
        read_w(stage, 1);
        __builtin_amdgcn_sched_barrier(0);           // the compiler would gather the products and then wait for all reads
#pragma unroll
        for (int j = 0; j < MI; ++j) {
            mma_column<T>(wf[0], xf[j], acc, j);
            read_x(stage, 1, j);
            __builtin_amdgcn_sched_barrier(0);
        }
        const int freed = stage;
#pragma unroll
        for (int j = 0; j < MI; ++j) {
            mma_column<T>(wf[1], xf[j], acc, j);
            if (j == EARLY) {
                wait_vmcnt<0>();
                pipeline_barrier();
                if constexpr (KIND == 1) {
                    address(nxt);
                    aim(nxt);
                }
                stage ^= 1;
                read_w(stage, 0);
#pragma unroll
                for (int k = 0; k <= EARLY; ++k) read_x(stage, 0, k);
            } else if (j > EARLY) {
                read_x(stage, 0, j);
                if constexpr (KIND < 2)
#pragma unroll
                    for (int i = (j - EARLY - 1) * N / SLOTS; i < (j - EARLY) * N / SLOTS; ++i) load(i, KIND == 0 ? step + 2 : 0, freed);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    for (int tile = walk.next; tile < walk.end; tile += walk.by) {
        issue(1, stage ^ 1);
        Tile nxt = {0, 0, 0, 0};                     // no tile: no rows, and loads of nothing
        if (tile + walk.by < walk.end) nxt = locate(tile + walk.by);
        f32x4_t acc[NI][MI];
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int j = 0; j < MI; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        for (int step = 0; step < steps - 2; ++step) run(std::integral_constant<int, 0>(), step, nxt, acc);
        run(std::integral_constant<int, 1>(), steps - 2, nxt, acc);
        run(std::integral_constant<int, 2>(), steps - 1, nxt, acc);
        constexpr int PART = STAGE / WAVES;
        store_tile<T, NI, MI, PART>(a, cur.e, cur.m0 + wm, cur.m1, cur.n0, wn, acc, smem + (stage ^ 1) * STAGE + wave * PART);
        pipeline_barrier();
        cur = nxt;
    }
    wait_vmcnt<0>();
#endif
}

// ---------------------------------------------------------------------------------------------------------------
// Large tiles, 16-bit types: 32 MI x 256 (MI = 8: 256 x 256), one workgroup of 2 x 4 waves a CU.  A wave's 128 x 64 sums fill 128
// accumulation registers; the products of a 64-byte half step of a CU are 1024 cycles of its matrix units, its fragment reads
// 768 and the loads into LDS 256 cycles of LDS, so everything that is not a product has to run beside the products: that is
// what the order below is for.  Measured on 32768 rows x 2048 x 4096: 1.22 PFLOP/s from memory and 1.34 when all rows lie in
// L2, where the large library product reaches 1.33; in one burst after the barrier the loads cost a tenth of it, a burst of
// fragment reads another.  Four stages of 64 bytes, which keep three steps on their way, measured slower (1.09, against
// 1.17 of two at that time): 64-byte requests to L2.
//
// The products of one row fragment with four weight fragments, sums in accumulation registers.  In assembly because the
// compiler, with 128 of them and 64 registers of fragments, writes products to other registers than it adds to and spills.
// The first instruction covers a vector write to an operand just before.
template <typename T>
__device__ __forceinline__ void mma_row(const u32x4_t (&w)[4], const u32x4_t& x, f32x4_t (&acc)[4]) {
#define FD_MFMA4(OP)                                                                                                   \
    asm volatile("s_nop 1\n" OP " %0, %4, %8, %0\n" OP " %1, %5, %8, %1\n" OP " %2, %6, %8, %2\n" OP " %3, %7, %8, %3"   \
                 : "+a"(acc[0]), "+a"(acc[1]), "+a"(acc[2]), "+a"(acc[3])                                              \
                 : "v"(w[0]), "v"(w[1]), "v"(w[2]), "v"(w[3]), "v"(x))
    if constexpr (__is_same(T, __bf16)) FD_MFMA4("v_mfma_f32_16x16x32_bf16");
    else FD_MFMA4("v_mfma_f32_16x16x32_f16");
#undef FD_MFMA4
}

// Waits until the last of those products can be read; the compiler does not see them.
__device__ __forceinline__ void settle(f32x4_t (&acc)[4]) {
    asm volatile("s_nop 15\ns_nop 15" : "+a"(acc[0]), "+a"(acc[1]), "+a"(acc[2]), "+a"(acc[3])::"memory");
}

// The results of a wave of the large tile (16 MI rows from m0 on, weight rows wn .. wn + 63): bias, activation, gate and
// rounding in registers, 16 rows at a time through the wave's 2 KB of LDS to 16-byte stores (N is a multiple of 8).
// The loads of the next tile's first two steps are awaited before the first store, so that no later wait for loads is
// one for stores.
template <typename T, int ACT, bool GATED, int MI>
__device__ __forceinline__ void store_wide(const ExpertArgs& a, int e, int m0, int m1, int n0, int wn, const f32x4_t (&acc)[MI][4], char* part) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    const int lane = opaque(threadIdx.x & 63), quad = lane >> 4, r = lane & 15;
    const int first = n0 + (GATED ? wn / 2 : wn);                   // output column of the wave
    f32x4_t b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        // gated: tiles 0 and 2 are of the first half, 1 and 3 of the second
        const int n = first + (GATED ? i >> 1 : i) * 16 + quad * 4;
        b[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        if (a.bias && n < a.N) {
            T raw[4];
            __builtin_memcpy(raw, (const T*)a.bias + (int64_t)e * a.wrows + (GATED && (i & 1) ? a.N : 0) + n, sizeof(raw));
#pragma unroll
            for (int c = 0; c < 4; ++c) b[i][c] = (float)raw[c];
        }
    }
    wait_vmcnt<0>();
    // a lane stores the 16-byte piece p of rows row0, row0 + ROWS, ..
    constexpr int PIECES = GATED ? 4 : 8, ROWS = 64 / PIECES;
    const int row0 = lane / PIECES, p = lane % PIECES, n = first + p * 8;
    T* out = (T*)a.y + (int64_t)(m0 + row0) * a.N + n;
#pragma unroll
    for (int j = 0; j < MI; ++j) {
#pragma unroll
        for (int i = 0; i < 4; i += GATED ? 2 : 1) {
            T4 q;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                float v = activate<T>(acc[j][i][c] + b[i][c], ACT);
                if (GATED) v *= acc[j][GATED ? i + 1 : i][c] + b[GATED ? i + 1 : i][c];
                q[c] = (T)v;
            }
            // 8 bytes at column i * 16 + quad * 4 (gated: i / 2 * 16): rows of PIECES pieces of 16 bytes, spread over the banks
            const int at = (GATED ? i / 2 : i) * 2 + (quad >> 1);
            *(T4*)(part + r * (PIECES * 16) + ((at ^ (GATED ? (r >> 2) & 3 : r & 7)) * 16) + (quad & 1) * 8) = q;
        }
        wave_fence();
#pragma unroll
        for (int h = 0; h < 16 / ROWS; ++h) {
            const int row = row0 + h * ROWS;
            const u32x4_t q = *(const u32x4_t*)(part + row * (PIECES * 16) + ((p ^ (GATED ? (row >> 2) & 3 : row & 7)) * 16));
            if (m0 + j * 16 + row < m1 && n < a.N) __builtin_memcpy(out + (int64_t)(j * 16 + h * ROWS) * a.N, &q, 16);
        }
        wave_fence();
    }
}

template <typename T, int ACT, bool GATED, int MI>
__global__ __launch_bounds__(512, 2) void expert_wide_kernel(ExpertArgs a, unsigned x_bytes) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int BM = 32 * MI, ROWS = 256, BN = 256, WN = 4, WAVES = 8, G = ROWS / 8 / WAVES, STAGE = (ROWS + BN) * 128;
    constexpr int NI = 4, EARLY = 1;
    constexpr unsigned NONE = 0x80000000u;
    // one array: the compiler waits for all loads into LDS before it reads an array of its own
    __shared__ __attribute__((aligned(16))) char smem[2 * STAGE + WAVES * 2048 + (FD_EXPERT_MAX + ROWS) * 4];
    int *ends = (int*)(smem + 2 * STAGE + WAVES * 2048), *list = ends + FD_EXPERT_MAX;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const TileScan scan = scan_tiles(a, BM, ends);
    zero_rest<T>(a, scan.routed);
    TileWalk walk = walk_tiles(scan, a);
    if (walk.next >= walk.end) return;
    const int row_bytes = a.K * (int)sizeof(T), pieces = row_bytes / 16, steps = (pieces + 7) / 8;
    // Lane l loads 16 bytes of row l / 8 of every 8-row load, the piece that goes to position l % 8.  (r >> 1) & 7 is
    // the same for all loads of a lane: they lie 8 * WAVES rows apart, and WAVES is even.
    const int lrow = wave * 8 + (lane >> 3), piece = (lane & 7) ^ ((lrow >> 1) & 7);

    struct Tile {
        int e, m0, m1, n0;
    };
    // which tile, and a request for its part of the row list, which goes to LDS like the rows
    auto locate = [&](int tile) {
        Tile t;
        locate_tile(scan, a, ends, BM, tile / a.tiles_n, t.e, t.m0, t.m1);
        t.n0 = (tile % a.tiles_n) * (a.gated ? BN / 2 : BN);
        if (a.rows && wave < ROWS / 64) {
            const __amdgpu_buffer_rsrc_t lr = __builtin_amdgcn_make_buffer_rsrc((void*)(a.rows + t.m0), 0, (unsigned)(t.m1 - t.m0) * 4, 0x00020000);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(lr, (__attribute__((address_space(3))) void*)(list + wave * 64), 4,
                                                     (wave * 64 + opaque(lane)) * 4, 0, 0, 0);
        }
        return t;
    };
    unsigned xo[G], wo[G];                      // byte offset of the lane's piece of step 0, NONE for no row
    auto address = [&](const Tile& t) {
        const int64_t limit = a.rows ? a.x_rows : ROWS;
        const int lrow = wave * 8 + (opaque(lane) >> 3);
#pragma unroll
        for (int i = 0; i < G; ++i) {
            const int r = lrow + WAVES * 8 * i, src = a.rows ? list[r] : r, row = weight_row(a, t.n0, r);
            xo[i] = src >= 0 && src < limit && t.m0 + r < t.m1 ? (unsigned)src * row_bytes + piece * 16 : NONE;
            wo[i] = row >= 0 && t.m0 < t.m1 ? (unsigned)row * row_bytes + piece * 16 : NONE;
        }
    };
    // what is loaded: a tile's rows and weights, their buffers, and whether the lane's piece of the step lies behind K
    __amdgpu_buffer_rsrc_t xr, wr;
    auto aim = [&](const Tile& t) {
        // without a row list the rows of a tile are a range of their own, so x may be of any size; a row at least, so that the
        // offset of a step never passes the end, which the range check subtracts it from
        xr = __builtin_amdgcn_make_buffer_rsrc((void*)((const char*)a.x + (a.rows ? 0 : (int64_t)t.m0 * row_bytes)), 0,
                                               a.rows ? x_bytes : (unsigned)max(t.m1 - t.m0, 1) * row_bytes, 0x00020000);
        wr = __builtin_amdgcn_make_buffer_rsrc((void*)((const char*)a.w + (int64_t)t.e * a.wrows * row_bytes), 0, (unsigned)a.wrows * row_bytes,
                                               0x00020000);
    };
    auto load = [&](int i, int step, int stage) {
        char* base = smem + stage * STAGE + wave * 1024;
        const bool none = step * 8 + piece >= pieces;
        if (i < G)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(xr, (__attribute__((address_space(3))) void*)(base + WAVES * i * 1024), 16,
                                                     none ? NONE : xo[i % G], step * 128, 0, 0);
        else
            __builtin_amdgcn_raw_ptr_buffer_load_lds(wr, (__attribute__((address_space(3))) void*)(base + ROWS * 128 + WAVES * (i - G) * 1024), 16,
                                                     none ? NONE : wo[i % G], step * 128, 0, 0);
    };
    auto issue = [&](int step, int stage) {
#pragma unroll
        for (int i = 0; i < 2 * G; ++i) load(i, step, stage);
    };
    const int wm = (wave / WN) * (BM / 2), wn = (wave % WN) * 64;
    const int frow = lane & 15, sw = (frow >> 1) & 7;
    int xf_off[2], wf_off[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int pos = ((h * 4 + (lane >> 4)) ^ sw) * 16;
        xf_off[h] = (wm + frow) * 128 + pos;
        wf_off[h] = (ROWS + wn + frow) * 128 + pos;
    }

    // One pipeline over all steps of all tiles.  Fragments are read half a step ahead: a row fragment is replaced by that
    // of the next half as soon as its products are issued, the weight fragments have two sets.  Early in the second
    // half, when all of the stage has been read, the next step's data is awaited and the stage goes to the load of the step
    // after next, the next tile's at a tile's last two steps.  The results have LDS of their own.
    u32x4_t xf[MI], wf[2][NI];
    auto read_x = [&](int stage, int h, int j) { xf[j] = *(const u32x4_t*)(smem + stage * STAGE + xf_off[h] + j * 2048); };
    auto read_w = [&](int stage, int h) {
#pragma unroll
        for (int i = 0; i < NI; ++i) wf[h][i] = *(const u32x4_t*)(smem + stage * STAGE + wf_off[h] + i * 2048);
    };
    Tile cur = locate(walk.next);
    wait_vmcnt<0>();
    pipeline_barrier();
    address(cur);
    aim(cur);
    issue(0, 0);
    issue(1, 1);
    wait_vmcnt<0>();
    pipeline_barrier();
    int stage = 0;
    // One step.  KIND 0 loads the current tile's step after next, KIND 1 (the last but one) the next tile's first, KIND 2 (the
    // last) its second.  The loads go out between the products; one burst would hold the products up.
    auto run = [&](auto kind, int step, const Tile& nxt, f32x4_t (&acc)[MI][NI]) {
        constexpr int KIND = decltype(kind)::value, SLOTS = MI - 1 - EARLY, N = 2 * G;
        read_w(stage, 1);
        __builtin_amdgcn_sched_barrier(0);           // the compiler would gather the products and then wait for all reads
#pragma unroll
        for (int j = 0; j < MI; ++j) {
            mma_row<T>(wf[0], xf[j], acc[j]);
            read_x(stage, 1, j);
            __builtin_amdgcn_sched_barrier(0);
        }
        const int freed = stage;
#pragma unroll
        for (int j = 0; j < MI; ++j) {
            mma_row<T>(wf[1], xf[j], acc[j]);
            if (j == EARLY) {
                if (step > 0) wait_vmcnt<0>();       // a tile's second step has been awaited before the stores of the tile before
                pipeline_barrier();
                if constexpr (KIND == 1) {
                    address(nxt);
                    aim(nxt);
                }
                stage ^= 1;
                if constexpr (KIND < 2) {
                    read_w(stage, 0);
#pragma unroll
                    for (int k = 0; k <= EARLY; ++k) read_x(stage, 0, k);
                }
            } else if (j > EARLY) {
                if constexpr (KIND < 2) read_x(stage, 0, j);
#pragma unroll
                for (int i = (j - EARLY - 1) * N / SLOTS; i < (j - EARLY) * N / SLOTS; ++i)
                    load(i, KIND == 0 ? step + 2 : KIND - 1, freed);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    for (int tile = walk.next; tile < walk.end; tile += walk.by) {
        Tile nxt = {0, 0, 0, 0};                     // no tile: no rows, and loads of nothing
        if (tile + walk.by < walk.end) nxt = locate(tile + walk.by);
        f32x4_t acc[MI][NI];
#pragma unroll
        for (int j = 0; j < MI; ++j)
#pragma unroll
            for (int i = 0; i < NI; ++i) acc[j][i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        read_w(stage, 0);
#pragma unroll
        for (int j = 0; j < MI; ++j) read_x(stage, 0, j);
        for (int step = 0; step < steps - 2; ++step) run(std::integral_constant<int, 0>(), step, nxt, acc);
        run(std::integral_constant<int, 1>(), steps - 2, nxt, acc);
        run(std::integral_constant<int, 2>(), steps - 1, nxt, acc);
#pragma unroll
        for (int j = 0; j < MI; ++j) settle(acc[j]);
        store_wide<T, ACT, GATED, MI>(a, cur.e, cur.m0 + wm, cur.m1, cur.n0, wn, acc, smem + 2 * STAGE + wave * 2048);
        cur = nxt;
    }
    wait_vmcnt<0>();
#endif
}

// ---------------------------------------------------------------------------------------------------------------
// Few rows an expert: the weights are the traffic and each is used once, so they go straight to registers, in any alignment.
// A workgroup owns 16 output columns of an expert (gated: 16 of each half) for up to 16 * MT of its rows; its WAVES waves take
// every WAVES-th 64-byte chunk of K, U chunks in flight each, and their sums meet in LDS, added in the order of the waves.
template <typename T, int MT, int G, int WAVES, int U>
__global__ __launch_bounds__(WAVES * 64) void expert_stream_kernel(ExpertArgs a) {
    constexpr int V = 16 / (int)sizeof(T), CHUNK = 4 * V;
    __shared__ f32x4_t part[WAVES][MT][G][64];
    __shared__ int ends[FD_EXPERT_MAX];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15;
    const TileScan scan = scan_tiles(a, 16 * MT, ends);
    zero_rest<T>(a, scan.routed);
    const TileWalk walk = walk_tiles(scan, a);
    const int full = a.K / CHUNK;
    for (int tile = walk.next; tile < walk.end; tile += walk.by) {
        int e, m0, m1;
        locate_tile(scan, a, ends, 16 * MT, tile / a.tiles_n, e, m0, m1);
        const int n0 = (tile % a.tiles_n) * 16;
        const T *wp[G], *xp[MT];
        bool none[MT];
#pragma unroll
        for (int g = 0; g < G; ++g) wp[g] = (const T*)a.w + ((int64_t)e * a.wrows + g * a.N + min(n0 + r, a.N - 1)) * a.K + (lane >> 4) * V;
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const int64_t row = source_row(a, min(m0 + t * 16 + r, m1 - 1));
            none[t] = row < 0;
            xp[t] = (a.x_rows ? (const T*)a.x + (row < 0 ? 0 : row) * a.K : (const T*)a.w) + (lane >> 4) * V;
        }
        f32x4_t acc[MT][G];
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int g = 0; g < G; ++g) acc[t][g] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        auto multiply = [&](const u32x4_t (&w)[G], u32x4_t (&x)[MT]) {
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                if (none[t]) x[t] = u32x4_t{0, 0, 0, 0};
#pragma unroll
                for (int g = 0; g < G; ++g) acc[t][g] = mma_piece<T>(w[g], x[t], acc[t][g]);
            }
        };
        int c = wave;
        for (; c + (U - 1) * WAVES < full; c += U * WAVES) {
            u32x4_t w[U][G], x[U][MT];
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
                for (int g = 0; g < G; ++g) __builtin_memcpy(&w[u][g], wp[g] + (int64_t)(c + u * WAVES) * CHUNK, 16);
#pragma unroll
                for (int t = 0; t < MT; ++t) __builtin_memcpy(&x[u][t], xp[t] + (int64_t)(c + u * WAVES) * CHUNK, 16);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) multiply(w[u], x[u]);
        }
        for (; c * CHUNK < a.K; c += WAVES) {
            const int left = a.K - c * CHUNK - (lane >> 4) * V;
            u32x4_t w[G], x[MT];
#pragma unroll
            for (int g = 0; g < G; ++g) w[g] = load_piece(wp[g] + (int64_t)c * CHUNK, left);
#pragma unroll
            for (int t = 0; t < MT; ++t) x[t] = load_piece(xp[t] + (int64_t)c * CHUNK, left);
            multiply(w, x);
        }
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int g = 0; g < G; ++g) part[wave][t][g][lane] = acc[t][g];
        __syncthreads();
        for (int i = threadIdx.x; i < MT * 256; i += WAVES * 64) {
            const int t = i >> 8, m = m0 + t * 16 + ((i >> 4) & 15), n = n0 + (i & 15);
            const int at = (((i >> 4) & 15) + 16 * ((i & 15) >> 2)) * 4 + (i & 3);
            float v[G];
#pragma unroll
            for (int g = 0; g < G; ++g) {
                v[g] = 0.f;
#pragma unroll
                for (int q = 0; q < WAVES; ++q) v[g] += ((const float*)part[q][t][g])[at];
            }
            if (m >= m1 || n >= a.N) continue;
            const T* bias = a.bias ? (const T*)a.bias + (int64_t)e * a.wrows + n : nullptr;
            float out = activate<T>(v[0] + (bias ? (float)bias[0] : 0.f), a.act);
            if constexpr (G == 2) out *= v[1] + (bias ? (float)bias[a.N] : 0.f);
            ((T*)a.y)[(int64_t)m * a.N + n] = (T)out;
        }
        __syncthreads();
    }
}

// Tiles of BM slots in the worst case: every group ends in a partial tile.
static int64_t worst_tiles(int slots, int experts, int bm) { return slots / bm + (experts < slots ? experts : slots); }

static double expert_flops(const ExpertArgs& a) { return 2.0 * a.slots * a.wrows * (double)a.K; }
template <typename T>
static double expert_bytes(const ExpertArgs& a) {
    return (double)sizeof(T) * ((double)a.experts * a.wrows * a.K + (double)a.x_rows * a.K + (double)a.slots * a.N);
}

// CUs of the current device, asked for once.
static int compute_units() {
    static std::atomic<int> known[64];
    int dev = 0, cus = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
    if ((cus = known[dev].load(std::memory_order_relaxed)) > 0) return cus;
    if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0) return 256;
    known[dev].store(cus, std::memory_order_relaxed);
    return cus;
}

// Workgroups for tiles of BM slots: as many as run at once, a multiple of the 8 XCDs; 0 with an error if the tiles cannot
// be counted in 31 bits.
static int tile_grid(const ExpertArgs& a, int bm, int per_cu) {
    const int64_t most = (int64_t)compute_units() * per_cu, tiles = worst_tiles(a.slots, a.experts, bm) * a.tiles_n;
    if (tiles >= (int64_t(1) << 31) - (1 << 20)) {
        set_error("fd_expert_linear: more than 2^31 - 2^20 tiles");
        return 0;
    }
    return (int)(((tiles < most ? tiles : most) + 7) / 8 * 8);
}

template <typename T, int BM, int BN, int D, int OCC>
static int launch_expert_tile(ExpertArgs a, hipStream_t stream) {
    a.tiles_n = ceil_div(a.N, a.gated ? BN / 2 : BN);
    const int grid = tile_grid(a, BM, OCC);
    if (!grid) return FD_ERR_LIMIT;
    ProfScope scope(stream, "expert_tile", expert_flops(a), expert_bytes<T>(a));
    hipLaunchKernelGGL((expert_tile_kernel<T, BM, BN, D, OCC>), dim3(grid), dim3(256), 0, stream, a);
    FD_LAUNCH_CHECK();
    return FD_OK;
}

template <typename T, int BM, int BN, int WM, int WN, int OCC>
static int launch_expert_dma(ExpertArgs a, hipStream_t stream) {
    a.tiles_n = ceil_div(a.N, a.gated ? BN / 2 : BN);
    const int grid = tile_grid(a, BM, OCC);
    if (!grid) return FD_ERR_LIMIT;
    ProfScope scope(stream, "expert_dma", expert_flops(a), expert_bytes<T>(a));
    hipLaunchKernelGGL((expert_dma_kernel<T, BM, BN, WM, WN, OCC>), dim3(grid), dim3(WM * WN * 64), 0, stream, a,
                       (unsigned)(a.x_rows * a.K * (int64_t)sizeof(T)));
    FD_LAUNCH_CHECK();
    return FD_OK;
}

template <typename T, int MI, int ACT>
static int launch_expert_wide(ExpertArgs a, hipStream_t stream) {
    a.tiles_n = ceil_div(a.N, a.gated ? 128 : 256);
    const int grid = tile_grid(a, 32 * MI, 1);
    if (!grid) return FD_ERR_LIMIT;
    const unsigned x_bytes = (unsigned)(a.x_rows * a.K * (int64_t)sizeof(T));
    ProfScope scope(stream, "expert_wide", expert_flops(a), expert_bytes<T>(a));
    if (a.gated) hipLaunchKernelGGL((expert_wide_kernel<T, ACT, true, MI>), dim3(grid), dim3(512), 0, stream, a, x_bytes);
    else hipLaunchKernelGGL((expert_wide_kernel<T, ACT, false, MI>), dim3(grid), dim3(512), 0, stream, a, x_bytes);
    FD_LAUNCH_CHECK();
    return FD_OK;
}

template <typename T, int MI>
static int launch_expert_wide(const ExpertArgs& a, hipStream_t stream) {
    switch (a.act) {
        case FD_ACT_RELU: return launch_expert_wide<T, MI, FD_ACT_RELU>(a, stream);
        case FD_ACT_SILU: return launch_expert_wide<T, MI, FD_ACT_SILU>(a, stream);
        case FD_ACT_GELU: return launch_expert_wide<T, MI, FD_ACT_GELU>(a, stream);
        default: return launch_expert_wide<T, MI, FD_ACT_NONE>(a, stream);
    }
}

template <typename T, int MT, int WAVES, int U>
static int launch_expert_stream(ExpertArgs a, hipStream_t stream) {
    a.tiles_n = ceil_div(a.N, 16);
    const int grid = tile_grid(a, 16 * MT, 32 / WAVES);
    if (!grid) return FD_ERR_LIMIT;
    ProfScope scope(stream, "expert_stream", expert_flops(a), expert_bytes<T>(a));
    if (a.gated) hipLaunchKernelGGL((expert_stream_kernel<T, MT, 2, WAVES, U>), dim3(grid), dim3(WAVES * 64), 0, stream, a);
    else hipLaunchKernelGGL((expert_stream_kernel<T, MT, 1, WAVES, U>), dim3(grid), dim3(WAVES * 64), 0, stream, a);
    FD_LAUNCH_CHECK();
    return FD_OK;
}

// Rows that start on 16-byte borders and whose offsets have 31 bits can be loaded straight into LDS, in two steps of 128
// bytes or more.
template <typename T>
static bool dma_rows(const ExpertArgs& a) {
    const int64_t row = (int64_t)a.K * sizeof(T), limit = int64_t(1) << 31;
    return a.x_rows > 0 && row % 16 == 0 && row > 128 && ((uintptr_t)a.x | (uintptr_t)a.w) % 16 == 0 && a.wrows * row < limit &&
           (a.rows ? a.x_rows : 256) * row < limit;
}

struct ExpertChoice {
    int (*launch)(const ExpertArgs&, hipStream_t);
    const char* name;              // of the kernel and its tile, for fd_expert_linear_kernel
};

// Which kernel, by sizes, type and alignment (times in bfloat16 unless said otherwise).  What each expert gets is known on the
// device only, so it goes by the average: 4096 slots on 1024 experts of 1024 x 1024 take 513 us spread evenly, 548 with shares of
// 1 / e, and 148 when one expert has them all, whose weights the stream kernel then reads once for every 16 rows (as the only
// expert of a call it takes large tiles, 15 us).
//
// The stream kernel for up to 4 rows an expert (20 slots on 8 experts of 2 x 1024 x 2048: 14.9 us, 32 x 64 tiles 16.2 us, 64 x 64
// 20.6; 512 slots on 64 experts of 2 x 512 x 1024: 34.9, 28.6, 28.3 us), in float32 up to 12 (80 slots on those 8: 39.5,
// 45, 63 us): the weights are the traffic.  Beyond that it is offered beside the tiles, with 16 or 32 rows at a time: it
// splits K over its waves, so it wins where there are few tiles (200 slots, 256 x 1024: 7.8 us with 16 rows, 10.5 with 32,
// 18.4 with 32 x 64 tiles; in float16 5.5, 6.6 and 8.3; 500 slots: 11.3, 11.0, 18.6 and 7.3, 6.9, 8.6; 800 slots: 18.0, 16.3,
// 18.7 and 10.7, 9.5, 8.7).  Its loads bound it, 0.055 us for each of a lane's loads in a step of 128 bytes of K, 0.145 for
// 16-bit rows off 16-byte borders.  Long rows have eight waves a workgroup (float32, the 20 slots: 31.9 us, with four 34.8).
//
// Tiles: a CU works through ceil(tiles / CUs) of them, and one step of 128 bytes of K costs a CU (with all CUs busy)
// 1.75, 1.48 and 1.34 us for 256, 224 and 192 x 256, 0.57 us for 128 x 128, 0.37 us for 64 x 128 and 0.27 us for 64 x 64, but a step
// of a tile is not shorter than its loads take; the large ones, alone on their CU, need another 3.5 to 4 us for their ends.
// Large tiles win on many rows an expert (32768 rows, 2048 x 4096: 1.22 PFLOP/s for 256 x 256, 0.93, 0.73 and 0.51 for the small
// ones), a little smaller ones when the last round of tiles is nearly empty (12000 slots on 8 experts of 2048 x 2048: 126 us
// with 256 rows, 113 with 224, 133 with 192; 8000 on 32 experts of 2 x 1024 x 1024: 71, 64, 60 us), small ones when an expert
// has few (1200 slots on 16 such experts: 29 us with 256 x 256, 21, 20 and 20 us).  The large ones take outputs in eights
// and three steps or more.
// Through registers, for rows that are not aligned, it is 1.15 us for 128 x 128, 0.45 for 64 x 64 and 0.33 for 32 x 64 (62682 slots,
// 1448 x 1001: 394 and 583 us for the first two; 2331 slots, 333 x 1001: 34, 16.5, 14.4 us, of which these costs,
// fitted to more steps and tiles, take the second; 41076 slots on 33 experts of 2 x 47 x 3191: 122, 146, 184 us).  32 x 64 through
// registers has the shortest step of a single tile and is offered for aligned rows too, 0.24 us a step (796 slots on 50 experts
// of 1547 x 832: 29.9 us, 64 x 64 33 to 36, 64 x 128 31.3; 320 on 8 experts of 2 x 1024 x 2048: 19.3, 21.0 us).  In float32 the
// matrix units are slow enough (1/16) that every tile reaches the same rate (126 TFLOP/s) and the smallest wastes the least.
template <typename T>
static ExpertChoice choose_expert(const ExpertArgs& a) {
    const int64_t groups = a.experts < a.slots ? a.experts : a.slots, row_bytes = (int64_t)a.K * sizeof(T);
    const int steps = ceil_div(row_bytes, 128), cus = compute_units();
    auto tiles_of = [&](int bm, int bn) {
        // a group ends in half a tile on average, a single one where it does
        const double rows = groups == 1 ? ceil_div(a.slots, bm) : a.slots / (double)bm + groups / 2.0;
        return rows * ceil_div(a.wrows, bn);
    };
    const ExpertChoice stream16 =
        row_bytes < 8192 ? ExpertChoice{[](const ExpertArgs& p, hipStream_t q) { return launch_expert_stream<T, 1, 4, 4>(p, q); }, "stream 16 rows, 4 waves"}
                         : ExpertChoice{[](const ExpertArgs& p, hipStream_t q) { return launch_expert_stream<T, 1, 8, 4>(p, q); }, "stream 16 rows, 8 waves"};
    if (a.slots <= (sizeof(T) == 4 ? 12 : 4) * groups) return stream16;
    double least = 0.0;
    ExpertChoice best = {nullptr, nullptr};
    // a step costs a CU `step` for each of its tiles but takes `load` at least; `ends`: a tile's start and end
    auto offer = [&](int bm, int bn, double step, double load, double ends, const ExpertChoice& choice) {
        const double rounds = ceil(tiles_of(bm, bn) / cus), cost = steps * fmax(rounds * step, load) + rounds * ends;
        if (!best.launch || cost < least) {
            least = cost;
            best = choice;
        }
    };
    const bool aligned = dma_rows<T>(a);
    const bool whole = sizeof(T) == 4 || (((uintptr_t)a.x | (uintptr_t)a.w) % 16 == 0 && row_bytes % 16 == 0);
    auto offer_stream = [&](int mt, const ExpertChoice& choice) {
        const double step = (whole ? 0.055 : 0.145) * (mt + (a.gated ? 2 : 1)), tiles = tiles_of(16 * mt, a.gated ? 32 : 16) / cus;
        // of several groups the number of tiles is an estimate, which ceil() would take at its word
        const double rounds = groups == 1 || tiles <= 1.0 ? ceil(tiles) : 0.5 * (tiles + ceil(tiles)), cost = steps * step * rounds + 0.7 * (mt - 1);
        if (!best.launch || cost < least) {
            least = cost;
            best = choice;
        }
    };
    offer_stream(1, stream16);
    offer_stream(2, {[](const ExpertArgs& p, hipStream_t q) { return launch_expert_stream<T, 2, 4, 4>(p, q); }, "stream 32 rows, 4 waves"});
    if constexpr (sizeof(T) == 4) {
        offer(32, 64, 0.30, 0.45, 0.3, {[](const ExpertArgs& p, hipStream_t q) { return launch_expert_tile<T, 32, 64, 2, 4>(p, q); }, "tile 32 x 64"});
        if (aligned) offer(64, 64, 0.50, 0.90, 0.3, {[](const ExpertArgs& p, hipStream_t q) { return launch_expert_dma<T, 64, 64, 2, 2, 4>(p, q); }, "dma 64 x 64"});
        else offer(64, 64, 0.55, 0.90, 0.3, {[](const ExpertArgs& p, hipStream_t q) { return launch_expert_tile<T, 64, 64, 2, 4>(p, q); }, "tile 64 x 64"});
    } else {
        offer(32, 64, aligned ? 0.24 : 0.33, aligned ? 0.27 : 0.36, 0.3, {[](const ExpertArgs& p, hipStream_t q) { return launch_expert_tile<T, 32, 64, 2, 4>(p, q); }, "tile 32 x 64"});
        if (!aligned) {
            offer(64, 64, 0.45, 0.45, 0.3, {[](const ExpertArgs& p, hipStream_t q) { return launch_expert_tile<T, 64, 64, 2, 4>(p, q); }, "tile 64 x 64"});
            offer(128, 128, 1.15, 1.15, 1.0, {[](const ExpertArgs& p, hipStream_t q) { return launch_expert_tile<T, 128, 128, 1, 2>(p, q); }, "tile 128 x 128"});
        } else {
            offer(64, 64, 0.27, 0.55, 0.3, {[](const ExpertArgs& p, hipStream_t q) { return launch_expert_dma<T, 64, 64, 2, 2, 4>(p, q); }, "dma 64 x 64"});
            offer(64, 128, 0.37, 0.72, 0.5, {[](const ExpertArgs& p, hipStream_t q) { return launch_expert_dma<T, 64, 128, 2, 2, 3>(p, q); }, "dma 64 x 128"});
            offer(128, 128, 0.57, 0.80, 1.0, {[](const ExpertArgs& p, hipStream_t q) { return launch_expert_dma<T, 128, 128, 2, 2, 2>(p, q); }, "dma 128 x 128"});
            if (a.N % 8 == 0 && row_bytes > 256) {
                offer(192, 256, 1.34, 1.34, 3.4, {[](const ExpertArgs& p, hipStream_t q) { return launch_expert_wide<T, 6>(p, q); }, "wide 192 x 256"});
                offer(224, 256, 1.48, 1.48, 3.6, {[](const ExpertArgs& p, hipStream_t q) { return launch_expert_wide<T, 7>(p, q); }, "wide 224 x 256"});
                offer(256, 256, 1.75, 1.75, 3.9, {[](const ExpertArgs& p, hipStream_t q) { return launch_expert_wide<T, 8>(p, q); }, "wide 256 x 256"});
            }
        }
    }
    return best;
}

// Checks the shape of a call and puts it into `a`, whose pointers and activation are still to be set.
static int expert_shape(ExpertArgs& a, int dtype, int64_t x_rows, int inner, int experts, int outputs, bool gather, int64_t slots, int gated) {
    FD_REQUIRE(valid_dtype(dtype), "fd_expert_linear: unknown element type");
    FD_REQUIRE(x_rows >= 0 && inner > 0 && experts > 0 && outputs > 0 && slots >= 0, "fd_expert_linear: bad shape");
    FD_REQUIRE(gather || x_rows == slots || slots == 0, "fd_expert_linear: without a row list every row of x is a slot (%lld rows, %lld slots)", (long long)x_rows,
               (long long)slots);
    if (slots >= (int64_t(1) << 31) - 1024 || experts > FD_EXPERT_MAX || inner > (1 << 24) || outputs > (1 << 24)) {
        set_error("fd_expert_linear: at most 2^31 - 1024 slots, %d experts, 2^24 inputs and outputs", FD_EXPERT_MAX);
        return FD_ERR_LIMIT;
    }
    a = ExpertArgs();
    a.x_rows = x_rows; a.K = inner; a.N = outputs; a.wrows = outputs * (gated ? 2 : 1); a.experts = experts; a.slots = (int)slots;
    a.gated = gated != 0;
    return FD_OK;
}

}  // namespace fd

extern "C" {

int fd_expert_linear(const void* x, int dtype, int64_t x_rows, int inner, const void* weight, int experts, int outputs, const int32_t* offsets,
                     const int32_t* rows, int64_t slots, const void* bias, int activation, int gated, void* y, void* stream) {
    fd::ExpertArgs a;
    FD_TRY(fd::expert_shape(a, dtype, x_rows, inner, experts, outputs, rows != nullptr, slots, gated));
    FD_REQUIRE(activation >= FD_ACT_NONE && activation <= FD_ACT_GELU, "fd_expert_linear: unknown activation");
    if (slots == 0) return FD_OK;
    FD_REQUIRE((x || x_rows == 0) && weight && offsets && y, "fd_expert_linear: NULL pointer");
    a.x = x; a.w = weight; a.bias = bias; a.y = y; a.offsets = offsets; a.rows = rows; a.act = activation;
    return fd::with_dtype(dtype, [&](auto t) { return fd::choose_expert<decltype(t)>(a).launch(a, fd::as_stream(stream)); });
}

const char* fd_expert_linear_kernel(const void* x, int dtype, int64_t x_rows, int inner, const void* weight, int experts, int outputs,
                                    const int32_t* rows, int64_t slots, int gated) {
    fd::ExpertArgs a;
    if (fd::expert_shape(a, dtype, x_rows, inner, experts, outputs, rows != nullptr, slots, gated) != FD_OK) return nullptr;
    if (slots == 0) return "";
    a.x = x; a.w = weight; a.rows = rows;
    const char* name = nullptr;
    fd::with_dtype(dtype, [&](auto t) {
        name = fd::choose_expert<decltype(t)>(a).name;
        return FD_OK;
    });
    return name;
}

}  // extern "C"
