// Matrix products grouped by expert: slot s of a row list sorted by expert multiplies the weights of its expert,
//
//   y[s, :] = act(x[rows[s], :] . w[e]^T + bias[e]),   offsets[e] <= s < offsets[e + 1],
//   gated:  y[s, n] = act(v[n]) * v[N + n],  v = x . w[e]^T + bias[e] over the expert's 2N weight rows.
//
// The groups are ragged and known on the device only.  The grid is sized for the worst case (every group ends in a
// partial tile); a wave finds its tile with one scan over the offsets in registers, and workgroups beyond the last tile
// leave.  Slots behind offsets[experts] form one more group, whose tiles are zeros.
//
// Weights are [N, K] and rows [*, K], both with K contiguous, so both operands of a 16 x 16 matrix instruction are 16-byte
// pieces along K: lane l holds row l & 15, piece l >> 4.  The weights are the first operand: a lane's four results are
// then four consecutive columns of one row of y.  float32 takes four 16x16x4 instructions over the same 16 bytes (the
// k of a lane's j-th float is the same for both operands, which is all the sum needs).  Sums are held in float32.
#include "fd_elem.h"

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
template <>
__device__ __forceinline__ f32x4_t mma<float>(u32x4_t a, u32x4_t b, f32x4_t c) {
    const f32x4_t fa = __builtin_bit_cast(f32x4_t, a), fb = __builtin_bit_cast(f32x4_t, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(fa[i], fb[i], c, 0, 0, 0);
    return c;
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

__device__ __forceinline__ float activate(float v, int act) {
    if (act == FD_ACT_RELU) return fmaxf(v, 0.f);
    if (act == FD_ACT_SILU) return v / (1.f + expf(-v));
    if (act == FD_ACT_GELU) return 0.5f * v * erfcf(-0.70710678118654752f * v);     // no cancellation for v << 0
    return v;
}

// The group and rows of tile `tile` when every group is cut into tiles of BM rows: expert e (experts = the unrouted rest),
// slots [m0, m1).  Every lane of the wave takes the same number of consecutive groups; ends are clamped to [0, slots] and
// never decrease, so any content of `offsets` stays in bounds.  False: there is no such tile.
__device__ __forceinline__ bool find_tile(const int32_t* offsets, int experts, int slots, int bm, int tile, int& e, int& m0, int& m1) {
    const int lane = threadIdx.x & 63, per = (experts + 64) / 64;
    int end = 0;
    for (int i = lane * per; i < (lane + 1) * per; ++i) end = max(end, i < experts ? min(offsets[i + 1], slots) : slots);
    int upto = end;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int v = __shfl_up(upto, d, 64);
        if (lane >= d) upto = max(upto, v);
    }
    int start = __shfl_up(upto, 1, 64);
    if (lane == 0) start = 0;
    int tiles = 0, at = start;
    for (int i = lane * per; i < (lane + 1) * per; ++i) {
        const int to = max(at, i < experts ? min(offsets[i + 1], slots) : slots);
        tiles += (to - at + bm - 1) / bm;
        at = to;
    }
    int sum = tiles;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int v = __shfl_up(sum, d, 64);
        if (lane >= d) sum += v;
    }
    int first = sum - tiles;
    const bool mine = tile >= first && tile < sum;
    const unsigned long long who = __ballot(mine);
    if (who == 0) return false;
    int fe = 0, f0 = 0, f1 = 0;
    if (mine) {
        at = start;
        for (int i = lane * per; i < (lane + 1) * per; ++i) {
            const int to = max(at, i < experts ? min(offsets[i + 1], slots) : slots);
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
    const int src = __ffsll((long long)who) - 1;
    e = __builtin_amdgcn_readlane(fe, src);
    m0 = __builtin_amdgcn_readlane(f0, src);
    m1 = __builtin_amdgcn_readlane(f1, src);
    return true;
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

// Four results of one row and four consecutive columns, from column n on.
template <typename T>
__device__ __forceinline__ void store4(const ExpertArgs& a, int64_t row, int n, const float (&v)[4]) {
    T* p = (T*)a.y + row * a.N + n;
    if (n + 4 <= a.N) {
        T raw[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) raw[i] = (T)v[i];
        __builtin_memcpy(p, raw, sizeof(raw));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n + i < a.N) p[i] = (T)v[i];
    }
}

// bias, activation and gate of the results of MFMA tiles (`second`: the second half's, gated only)
template <typename T>
__device__ __forceinline__ void finish4(const ExpertArgs& a, int e, int64_t row, int n, const f32x4_t& first, const f32x4_t& second) {
    const T* bias = a.bias ? (const T*)a.bias + (int64_t)e * a.wrows : nullptr;
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bool in = n + i < a.N;
        float g = first[i] + (bias && in ? (float)bias[n + i] : 0.f);
        v[i] = activate(g, a.act);
        if (a.gated) v[i] *= second[i] + (bias && in ? (float)bias[a.N + n + i] : 0.f);
    }
    store4<T>(a, row, n, v);
}

// ---------------------------------------------------------------------------------------------------------------
// Tile kernel: BM slots x BN weight rows, 4 waves of (BM/2) x (BN/2), 128 bytes of K a step.  A row of a step is 8
// pieces; piece c of row r lies at c ^ ((r >> 1) & 7), which spreads the fragment reads over the LDS banks.
template <typename T, int BM, int BN>
__global__ __launch_bounds__(256, 2) void expert_tile_kernel(ExpertArgs a) {
    constexpr int V = 16 / (int)sizeof(T), BK = 8 * V;
    constexpr int RA = BM / 32, RB = BN / 32, MI = BM / 32, NI = BN / 32;
    __shared__ u32x4_t xs[BM * 8], ws[BN * 8];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int tile_n = blockIdx.x % a.tiles_n;
    int e, m0, m1;
    if (!find_tile(a.offsets, a.experts, a.slots, BM, blockIdx.x / a.tiles_n, e, m0, m1)) return;
    const int n0 = tile_n * (a.gated ? BN / 2 : BN);
    if (e == a.experts) {
        const int n1 = min(a.N, n0 + (a.gated ? BN / 2 : BN));
        for (int i = tid; i < (m1 - m0) * (n1 - n0); i += 256)
            ((T*)a.y)[(int64_t)(m0 + i / (n1 - n0)) * a.N + n0 + i % (n1 - n0)] = (T)0.f;
        return;
    }
    const int c = tid & 7, r0 = tid >> 3;
    const T *xp[RA], *wp[RB];
#pragma unroll
    for (int i = 0; i < RA; ++i) {
        const int s = m0 + r0 + 32 * i;
        const int64_t r = s < m1 ? source_row(a, s) : -1;
        xp[i] = r < 0 ? nullptr : (const T*)a.x + r * a.K;
    }
#pragma unroll
    for (int i = 0; i < RB; ++i) {
        const int r = weight_row(a, n0, r0 + 32 * i);
        wp[i] = r < 0 ? nullptr : (const T*)a.w + ((int64_t)e * a.wrows + r) * a.K;
    }
    f32x4_t acc[NI][MI];
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < MI; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};

    u32x4_t xr[RA], wr[RB];
    auto fetch = [&](int k) {
        const int at = k + c * V;
#pragma unroll
        for (int i = 0; i < RA; ++i) xr[i] = load_piece(xp[i] + at, xp[i] ? a.K - at : 0);
#pragma unroll
        for (int i = 0; i < RB; ++i) wr[i] = load_piece(wp[i] + at, wp[i] ? a.K - at : 0);
    };
    const int wm = (wave >> 1) * (BM / 2), wn = (wave & 1) * (BN / 2);
    fetch(0);
    for (int k = 0; k < a.K; k += BK) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < RA; ++i) {
            const int r = r0 + 32 * i;
            xs[r * 8 + (c ^ ((r >> 1) & 7))] = xr[i];
        }
#pragma unroll
        for (int i = 0; i < RB; ++i) {
            const int r = r0 + 32 * i;
            ws[r * 8 + (c ^ ((r >> 1) & 7))] = wr[i];
        }
        __syncthreads();
        if (k + BK < a.K) fetch(k + BK);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            u32x4_t xf[MI], wf[NI];
            const int piece = h * 4 + (lane >> 4);
#pragma unroll
            for (int j = 0; j < MI; ++j) {
                const int r = wm + j * 16 + (lane & 15);
                xf[j] = xs[r * 8 + (piece ^ ((r >> 1) & 7))];
            }
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int r = wn + i * 16 + (lane & 15);
                wf[i] = ws[r * 8 + (piece ^ ((r >> 1) & 7))];
            }
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int j = 0; j < MI; ++j) acc[i][j] = mma<T>(wf[i], xf[j], acc[i][j]);
        }
    }
#pragma unroll
    for (int j = 0; j < MI; ++j) {
        const int s = m0 + wm + j * 16 + (lane & 15);
        if (s >= m1) continue;
        if (a.gated) {
#pragma unroll
            for (int i = 0; i < NI; i += 2) {
                const int n = n0 + (wn + i * 16) / 2 + 4 * (lane >> 4);
                if (n < a.N) finish4<T>(a, e, s, n, acc[i][j], acc[i + 1][j]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int n = n0 + wn + i * 16 + 4 * (lane >> 4);
                if (n < a.N) finish4<T>(a, e, s, n, acc[i][j], acc[i][j]);
            }
        }
    }
}

// Tiles of BM slots in the worst case: every group (the unrouted rest is one more) ends in a partial tile.
static int64_t worst_tiles(int slots, int experts, int bm) {
    return slots / bm + (experts + 1 < slots ? experts + 1 : slots);
}

template <typename T, int BM, int BN>
static int launch_expert_tile(ExpertArgs a, hipStream_t stream) {
    a.tiles_n = ceil_div(a.N, a.gated ? BN / 2 : BN);
    const int64_t blocks = worst_tiles(a.slots, a.experts, BM) * a.tiles_n;
    if (blocks >= (int64_t(1) << 31)) {
        set_error("fd_expert_linear: too many tiles");
        return FD_ERR_LIMIT;
    }
    hipLaunchKernelGGL((expert_tile_kernel<T, BM, BN>), dim3((unsigned)blocks), dim3(256), 0, stream, a);
    FD_LAUNCH_CHECK();
    return FD_OK;
}

}  // namespace fd

extern "C" {

int fd_expert_linear(const void* x, int dtype, int64_t x_rows, int inner, const void* weight, int experts, int outputs, const int32_t* offsets,
                     const int32_t* rows, int64_t slots, const void* bias, int activation, int gated, void* y, void* stream) {
    FD_REQUIRE(fd::valid_dtype(dtype), "fd_expert_linear: unknown element type");
    FD_REQUIRE(x_rows >= 0 && inner > 0 && experts > 0 && outputs > 0 && slots >= 0, "fd_expert_linear: bad shape");
    FD_REQUIRE(activation >= FD_ACT_NONE && activation <= FD_ACT_GELU, "fd_expert_linear: unknown activation");
    FD_REQUIRE(rows || x_rows == slots, "fd_expert_linear: without a row list every row of x is a slot (%lld rows, %lld slots)", (long long)x_rows,
               (long long)slots);
    if (slots >= (int64_t(1) << 31) - 1024 || experts > FD_EXPERT_MAX || inner > (1 << 24) || outputs > (1 << 24)) {
        fd::set_error("fd_expert_linear: at most 2^31 - 1024 slots, %d experts, 2^24 inputs and outputs", FD_EXPERT_MAX);
        return FD_ERR_LIMIT;
    }
    if (slots == 0) return FD_OK;
    FD_REQUIRE((x || x_rows == 0) && weight && offsets && y, "fd_expert_linear: NULL pointer");
    fd::ExpertArgs a;
    a.x = x; a.w = weight; a.bias = bias; a.y = y; a.offsets = offsets; a.rows = rows; a.x_rows = x_rows;
    a.K = inner; a.N = outputs; a.wrows = outputs * (gated ? 2 : 1); a.experts = experts; a.slots = (int)slots; a.act = activation;
    a.gated = gated != 0; a.tiles_n = 0;
    const double s = fd::dtype_bytes(dtype);
    fd::ProfScope scope(fd::as_stream(stream), "expert_linear", 2.0 * slots * a.wrows * (double)inner,
                        s * ((double)experts * a.wrows * inner + (double)x_rows * inner + (double)slots * outputs));
    return fd::with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        if (slots < 64ll * experts) return fd::launch_expert_tile<T, 64, 64>(a, fd::as_stream(stream));
        return fd::launch_expert_tile<T, 128, 128>(a, fd::as_stream(stream));
    });
}

}  // extern "C"
