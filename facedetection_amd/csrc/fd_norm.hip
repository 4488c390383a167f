// Norms around a residual block, with the block's gate, residual scale and (for a block of experts) the weighted
// sum of a row's expert outputs; and that sum on its own.
//
//   h[t]  = sum_j weights[t,j] * y[slots[t,j]]            (expert blocks; otherwise h is read as it is)
//   x'[t] = x[t] + scale * act(gate) * norm(h[t])
//   u[t]  = norm(x'[t])
//   norm(v) = (v - mean) / sqrt(mean((v - mean)^2) + eps) * weight + bias,  mean = 0 for the RMS form
//
// Bound by memory: a row is read once, held in registers as float32 through all of this, and written once.  Means and
// squares are summed in float32 over the registers (two passes, no E[v^2] - mean^2), so the only rounding to the
// tensors' type is the one at the store; u is computed from the unrounded x'.  Measured: x float32 and h bfloat16, gate,
// both norms, 8160 x 1024: 25 us for 100 MB; two choices a row, bfloat16, 6000 x 2048: 31 us for 123 MB, where a large copy
// takes 21 and 26; the sum alone, 130560 x 1024 with two choices: 134 us for 0.8 GB.
#include "fd_elem.h"

namespace fd {

struct NormArgs {
    const void *x, *h, *gate;
    const float *post_weight, *post_bias, *pre_weight, *pre_bias, *weights;
    const int32_t* slots;
    void *x_out, *u;
    int64_t rows, h_rows;
    int width, k, rows_per_gate, gate_f32, gate_act, layer;
    float scale, eps;
};

__device__ __forceinline__ float gate_value(float g, int act) {
    // off by less than 12 * 2^-24 of the value; zero from g = -87.3 on, where it is below 2^-126
    if (act == FD_GATE_SIGMOID) return __builtin_amdgcn_rcpf(1.f + exp_fast(-g));
    if (act == FD_GATE_TANH) return tanhf(g);
    return g;
}

// Sum over the G lanes that share a row; every lane gets it.  G = 256 goes through LDS, alternating between two sets
// of words so that one barrier a sum is enough.
template <int G>
__device__ __forceinline__ float row_sum(float v, float (*part)[4], int& turn) {
#pragma unroll
    for (int d = (G < 64 ? G : 64) / 2; d > 0; d >>= 1) v += __shfl_xor(v, d, 64);
    if (G == 256) {
        if ((threadIdx.x & 63) == 0) part[turn][threadIdx.x >> 6] = v;
        __syncthreads();
        v = (part[turn][0] + part[turn][1]) + (part[turn][2] + part[turn][3]);
        turn ^= 1;
    }
    return v;
}

// The pieces of a lane: piece c has P elements from column at[c] on, and those before own[c] belong to another lane.  Pieces lie
// G * P apart; one that would end behind the row (of P elements or more) is moved back to the row's last P.  It then
// computes, and writes, the same values for the columns that it shares, and leaves them out of sums; whole pieces without a
// branch keep all loads of a row on their way at once (with partial pieces read element by element: 101351 x 947 in
// bfloat16 148 us).
template <int NC>
struct Pieces {
    int at[NC], own[NC];
    bool whole;                // every piece lies in the row
};

template <int G, int NC, int P>
__device__ __forceinline__ Pieces<NC> row_pieces(int lane, int width) {
    Pieces<NC> q;
    q.whole = width == G * NC * P;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int col = (c * G + lane) * P;
        q.at[c] = min(col, width - P);
        q.own[c] = min(col - q.at[c], P);
    }
    return q;
}

template <int NC, int P>
__device__ __forceinline__ float own_sum(const float (&v)[NC][P], const Pieces<NC>& q, bool square) {
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const float e = q.whole || i >= q.own[c] ? v[c][i] : 0.f;
            s = square ? fmaf(e, e, s) : s + e;
        }
    return s;
}

// weight and bias of a lane's pieces
template <int NC, int P>
struct NormParams {
    float weight[NC][P], bias[NC][P];
};

template <int NC, int P>
__device__ __forceinline__ void load_params(NormParams<NC, P>& p, const float* weight, const float* bias, const Pieces<NC>& q) {
#pragma unroll
    for (int c = 0; c < NC; ++c) load_whole<P>(weight + q.at[c], p.weight[c]);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        if (bias) load_whole<P>(bias + q.at[c], p.bias[c]);
        else
#pragma unroll
            for (int i = 0; i < P; ++i) p.bias[c][i] = 0.f;
    }
}

template <int G, int NC, int P>
__device__ __forceinline__ void normalise(float (&v)[NC][P], const NormParams<NC, P>& p, const Pieces<NC>& q, const NormArgs& a, float (*part)[4],
                                          int& turn) {
    if (a.layer) {
        const float mean = row_sum<G>(own_sum(v, q, false), part, turn) / (float)a.width;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int i = 0; i < P; ++i) v[c][i] -= mean;
    }
    const float r = rsqrtf(row_sum<G>(own_sum(v, q, true), part, turn) / (float)a.width + a.eps);
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int i = 0; i < P; ++i) v[c][i] = v[c][i] * r * p.weight[c][i] + p.bias[c][i];
}

// The index of a workgroup, and the grid for `blocks` of them: a grid dimension holds fewer than 2^32 threads.
constexpr int64_t GRID_BLOCKS = 1 << 23;
inline dim3 block_grid(int64_t blocks, int columns = 1) {
    const int64_t x = blocks < GRID_BLOCKS ? blocks : GRID_BLOCKS;
    return dim3((unsigned)x, columns, (unsigned)((blocks + x - 1) / x));
}
__device__ __forceinline__ int64_t block_index() { return (int64_t)blockIdx.z * gridDim.x + blockIdx.x; }

// Two of a row's choices, so that both are asked for before either is waited for; -1 for a choice that is not made.
struct ChoicePair {
    int32_t slot[2];
    float weight[2];
};

__device__ __forceinline__ ChoicePair choice_pair(const int32_t* slots, const float* weights, int k, int j, int64_t rows) {
    ChoicePair p;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const int at = j + q < k ? j + q : j;
        p.slot[q] = slots[at];
        p.weight[q] = weights[at];
        if (j + q >= k || p.slot[q] < 0 || p.slot[q] >= rows) p.slot[q] = -1;
    }
    return p;
}

// G lanes hold a row, NE elements each.  A piece is 16 bytes of x, 4 elements of a float32 x and 8 otherwise, so that neighbouring
// lanes read neighbouring pieces; rows shorter than that are read one by one (P = 1).  With 8 elements a lane there are
// registers to ask for everything that the row needs before the first sum is waited for.
template <typename TX, typename TH, int G, int NE, int P>
__global__ __launch_bounds__(256) void residual_norm_kernel(NormArgs a) {
    constexpr int NC = NE / P;
    constexpr bool AHEAD = NE == 8;
    __shared__ float part[2][4];
    int turn = 0;
    const int lane = threadIdx.x % G;
    const int64_t row = block_index() * (256 / G) + threadIdx.x / G;
    if (row >= a.rows) return;                       // a whole group of G lanes: G = 256 never leaves early
    const Pieces<NC> q = row_pieces<G, NC, P>(lane, a.width);
    const int64_t start = row * a.width, gate_row = a.gate ? (row / a.rows_per_gate) * a.width : 0;
    float x[NC][P], h[NC][P], gate[NC][P];
#pragma unroll
    for (int c = 0; c < NC; ++c) load_whole<P>((const TX*)a.x + start + q.at[c], x[c]);
    if (a.h && !a.slots)
#pragma unroll
        for (int c = 0; c < NC; ++c) load_whole<P>((const TH*)a.h + start + q.at[c], h[c]);
    NormParams<NC, P> post, pre;
    auto load_gate = [&](int c) {
        if (a.gate_f32) load_whole<P>((const float*)a.gate + gate_row + q.at[c], gate[c]);
        else load_whole<P>((const TH*)a.gate + gate_row + q.at[c], gate[c]);
    };
    if (AHEAD) {
        if (a.post_weight) load_params(post, a.post_weight, a.post_bias, q);
        if (a.pre_weight) load_params(pre, a.pre_weight, a.pre_bias, q);
        if (a.gate)
#pragma unroll
            for (int c = 0; c < NC; ++c) load_gate(c);
    }
    if (a.h) {
        if (a.slots) {
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int i = 0; i < P; ++i) h[c][i] = 0.f;
            for (int j = 0; j < a.k; j += 2) {
                const ChoicePair p = choice_pair(a.slots + row * a.k, a.weights + row * a.k, a.k, j, a.h_rows);
#pragma unroll
                for (int s = 0; s < 2; ++s)
                    if (p.slot[s] >= 0)
#pragma unroll
                        for (int c = 0; c < NC; ++c) {
                            float y[P];
                            load_whole<P>((const TH*)a.h + (int64_t)p.slot[s] * a.width + q.at[c], y);
#pragma unroll
                            for (int i = 0; i < P; ++i) h[c][i] += p.weight[s] * y[i];
                        }
            }
        }
        if (a.post_weight) {
            if (!AHEAD) load_params(post, a.post_weight, a.post_bias, q);
            normalise<G, NC, P>(h, post, q, a, part, turn);
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            if (a.gate) {
                if (!AHEAD) load_gate(c);
#pragma unroll
                for (int i = 0; i < P; ++i) h[c][i] *= gate_value(gate[c][i], a.gate_act);
            }
#pragma unroll
            for (int i = 0; i < P; ++i) x[c][i] += a.scale * h[c][i];
            if (q.own[c] < P) store_whole<P>((TX*)a.x_out + start + q.at[c], x[c]);
        }
    }
    if (a.pre_weight) {
        if (!AHEAD) load_params(pre, a.pre_weight, a.pre_bias, q);
        normalise<G, NC, P>(x, pre, q, a, part, turn);
#pragma unroll
        for (int c = 0; c < NC; ++c)
            if (q.own[c] < P) store_whole<P>((TH*)a.u + start + q.at[c], x[c]);
    }
}

template <typename TX, typename TH>
static int launch_residual_norm(const NormArgs& a, hipStream_t stream) {
    // Lanes per row: 16 up to 256 (100000 x 256 in bfloat16: 17.8 us, a wave a row 30.9); 8 elements a lane up to 512 and,
    // with a block's output, in a workgroup's reach of 2048 (50000 rows of 2048 in bfloat16: 163 us, a wave a row 203; 6000
    // with two choices: 27 and 33 us).  A wave for up to 1024 (101351 x 947: 94 us, two waves 130) and for the norm alone up
    // to 2048 (50000 x 1900: 92 us, a workgroup 109), unless there are too few rows to give every CU eight waves.
    constexpr int P = 16 / (int)sizeof(TX);
    const bool few = a.rows < 2048;
#define FD_NORM(G, NE, PIECE)                                                                                               \
    do {                                                                                                                    \
        const int64_t blocks = (a.rows + 256 / G - 1) / (256 / G);                                                          \
        hipLaunchKernelGGL((residual_norm_kernel<TX, TH, G, NE, PIECE>), block_grid(blocks), dim3(256), 0, stream, a);      \
    } while (0)
    if (a.width < P) FD_NORM(16, 8, 1);
    else if (a.width <= 128) FD_NORM(16, 8, P);
    else if (a.width <= 256) FD_NORM(16, 16, P);
    else if (a.width <= 512) FD_NORM(64, 8, P);
    else if (a.width <= 1024 && !few) FD_NORM(64, 16, P);
    else if (a.width <= 2048 && !few && !a.h) FD_NORM(64, 32, P);
    else if (a.width <= 2048) FD_NORM(256, 8, P);
    else if (a.width <= 4096) FD_NORM(256, 16, P);
    else if (a.width <= 8192) FD_NORM(256, 32, P);
    else FD_NORM(256, 64, P);
#undef FD_NORM
    FD_LAUNCH_CHECK();
    return FD_OK;
}

// out[t] = sum_j weights[t,j] * y[slots[t,j]], terms in the order of j.  A thread owns P columns of a row; the last piece of a
// row is moved back to lie in it, and writes the columns that it shares a second time.
template <typename T, int P>
__global__ __launch_bounds__(256) void expert_combine_kernel(const T* y, int64_t y_rows, int width, const int32_t* slots, const float* weights,
                                                             int64_t rows, int k, T* out) {
    const int64_t row = block_index() * blockDim.y + threadIdx.y;
    if (row >= rows) return;
    // unsigned: a width is below 2^31 and a stride at most 2^16 * 2^8 * 8, so the column behind the last one still has 32 bits
    const unsigned columns = width, stride = gridDim.y * blockDim.x * P;
    for (unsigned col = (blockIdx.y * blockDim.x + threadIdx.x) * P; col < columns; col += stride) {
        const unsigned at = min(col, columns - P);
        float acc[P];
#pragma unroll
        for (int i = 0; i < P; ++i) acc[i] = 0.f;
        for (int j = 0; j < k; j += 2) {
            const ChoicePair p = choice_pair(slots + row * k, weights + row * k, k, j, y_rows);
            float v[2][P];
#pragma unroll
            for (int s = 0; s < 2; ++s)
                if (p.slot[s] >= 0) load_whole<P>(y + (int64_t)p.slot[s] * width + at, v[s]);
#pragma unroll
            for (int s = 0; s < 2; ++s)
                if (p.slot[s] >= 0)
#pragma unroll
                    for (int i = 0; i < P; ++i) acc[i] += p.weight[s] * v[s][i];
        }
        store_whole<P>(out + row * width + at, acc);
    }
}

}  // namespace fd

extern "C" {

int fd_residual_norm(const fd_norm_args* p, void* stream) {
    FD_REQUIRE(p, "fd_residual_norm: args is NULL");
    FD_REQUIRE(fd::valid_dtype(p->x_dtype) && fd::valid_dtype(p->h_dtype), "fd_residual_norm: unknown element type");
    FD_REQUIRE(p->x_dtype == p->h_dtype || p->x_dtype == FD_F32, "fd_residual_norm: x is float32 or of the block's type");
    FD_REQUIRE(p->rows >= 0 && p->width > 0, "fd_residual_norm: bad shape [%lld, %d]", (long long)p->rows, p->width);
    if (p->width > FD_NORM_MAX_WIDTH) {
        fd::set_error("fd_residual_norm: rows of %d elements; at most %d are held in registers", p->width, FD_NORM_MAX_WIDTH);
        return FD_ERR_LIMIT;
    }
    FD_REQUIRE(p->rows < (int64_t(1) << 31), "fd_residual_norm: too many rows");
    if (p->rows == 0) return FD_OK;
    FD_REQUIRE(p->x, "fd_residual_norm: x is NULL");
    // an empty h has no address; with slots it is there all the same, and every slot lies outside of it
    const void* h = p->h ? p->h : (p->slots && p->h_rows == 0 ? p->x : nullptr);
    FD_REQUIRE(h ? p->x_out != nullptr : p->pre_weight != nullptr, "fd_residual_norm: no output asked for");
    FD_REQUIRE(!p->pre_weight || p->u, "fd_residual_norm: u is NULL");
    FD_REQUIRE(h || !(p->post_weight || p->gate || p->slots), "fd_residual_norm: post norm, gate and slots belong to h");
    FD_REQUIRE(!p->post_bias || p->post_weight, "fd_residual_norm: post_bias without post_weight");
    FD_REQUIRE(!p->pre_bias || p->pre_weight, "fd_residual_norm: pre_bias without pre_weight");
    FD_REQUIRE(!p->slots || (p->weights && p->k > 0 && p->h_rows >= 0), "fd_residual_norm: slots need weights and k > 0");
    FD_REQUIRE(!p->gate || (p->gate_rows > 0 && p->rows % p->gate_rows == 0), "fd_residual_norm: %lld gate rows do not divide %lld rows",
               (long long)p->gate_rows, (long long)p->rows);
    FD_REQUIRE(!p->gate || p->gate_dtype == FD_F32 || p->gate_dtype == p->h_dtype, "fd_residual_norm: gate is float32 or of the block's type");
    FD_REQUIRE(p->gate_act >= FD_GATE_NONE && p->gate_act <= FD_GATE_TANH, "fd_residual_norm: unknown gate activation");
    FD_REQUIRE(p->eps > 0.f, "fd_residual_norm: eps must be positive");
    fd::NormArgs a;
    a.x = p->x; a.h = h; a.gate = p->gate;
    a.post_weight = p->post_weight; a.post_bias = p->post_bias; a.pre_weight = p->pre_weight; a.pre_bias = p->pre_bias;
    a.weights = p->weights; a.slots = p->slots; a.x_out = p->x_out; a.u = p->u;
    a.rows = p->rows; a.h_rows = p->slots ? p->h_rows : p->rows; a.width = p->width; a.k = p->k;
    a.rows_per_gate = p->gate ? (int)(p->rows / p->gate_rows) : 1;
    a.gate_f32 = p->gate_dtype == FD_F32; a.gate_act = p->gate_act; a.layer = p->layer != 0; a.scale = p->scale; a.eps = p->eps;
    const double n = (double)p->rows * p->width;
    const int sx = fd::dtype_bytes(p->x_dtype), sh = fd::dtype_bytes(p->h_dtype);
    fd::ProfScope scope(fd::as_stream(stream), "residual_norm", n * 8,
                        n * (sx + (h ? sx + sh * (p->slots ? p->k : 1) : 0) + (p->u ? sh : 0)));
    return fd::with_dtype(p->h_dtype, [&](auto th) {
        using TH = decltype(th);
        return p->x_dtype == p->h_dtype ? fd::launch_residual_norm<TH, TH>(a, fd::as_stream(stream))
                                        : fd::launch_residual_norm<float, TH>(a, fd::as_stream(stream));
    });
}

int fd_expert_combine(const void* y, int dtype, int64_t y_rows, int width, const int32_t* slots, const float* weights, int64_t rows, int k,
                      void* out, void* stream) {
    FD_REQUIRE(fd::valid_dtype(dtype), "fd_expert_combine: unknown element type");
    FD_REQUIRE(rows >= 0 && rows < (int64_t(1) << 31) && y_rows >= 0 && width > 0 && k > 0, "fd_expert_combine: bad shape");
    if (rows == 0) return FD_OK;
    FD_REQUIRE(slots && weights && out && (y || y_rows == 0), "fd_expert_combine: NULL pointer");
    const int per = width < 8 ? 1 : 8, pieces = fd::ceil_div(width, per);
    int bx = 1;
    while (bx < pieces && bx < 256) bx *= 2;
    const dim3 block(bx, 256 / bx);
    const int gy = fd::ceil_div(pieces, bx);
    const dim3 grid = fd::block_grid((rows + block.y - 1) / block.y, gy < 65535 ? gy : 65535);
    const double n = (double)rows * width * fd::dtype_bytes(dtype);
    fd::ProfScope scope(fd::as_stream(stream), "expert_combine", 2.0 * rows * width * k, n * (k + 1));
    return fd::with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        if (per == 1)
            hipLaunchKernelGGL((fd::expert_combine_kernel<T, 1>), grid, block, 0, fd::as_stream(stream), (const T*)y, y_rows, width, slots, weights,
                               rows, k, (T*)out);
        else
            hipLaunchKernelGGL((fd::expert_combine_kernel<T, 8>), grid, block, 0, fd::as_stream(stream), (const T*)y, y_rows, width, slots, weights,
                               rows, k, (T*)out);
        FD_LAUNCH_CHECK();
        return FD_OK;
    });
}

}  // extern "C"
