// Route of rows to experts: the k largest logits of a row, their softmax weights, and the stable counting sort of
// all choices by expert that lays the rows out for the grouped products (fd_expert_linear).
//
//   choice order: logit descending, then expert ascending; -inf, NaN and masked rows choose nothing
//   weights[t,j] = exp(l_j - l_0) / sum, the sum over the row's choices (normalize) or over all its experts
//   slots[t,j]   = position of the choice among all choices sorted by (expert, t);  rows[slots[t,j]] = t
//
// Bound by the read of the logits, with the walk close behind it (130560 rows of 64 float32 logits, 4 choices of a softmax
// over all, with mask: 23.2 us in all for 42 MB; a trace has 18.5 us for this launch and 6.4 for the second).  Two threads share
// a row: each walks its half of every 32 experts through LDS
// (staged by coalesced loads, 33 words a row so that the walk has no bank conflicts) and keeps its k best in registers; the
// first thread then takes the other's in.  Where the rows are too few for that, a wave takes one.  A row's experts are
// distinct, so the rank of a choice among its workgroup's choices of that expert is a population count over one bit per row:
// set with LDS atomics, whose order does not show.  Workgroups are joined by a second launch that sums their counts; where
// there are many, whose sums would grow with the square of the rows, by a third between the two that scans them.
#include "fd_elem.h"

namespace fd {

constexpr int ROUTE_ROWS = 512;            // rows of a workgroup; two threads a row choose, one places
constexpr int ROUTE_COLS = 32;             // experts staged at a time
constexpr int ROUTE_WORDS = ROUTE_ROWS / 64;
constexpr int ROUTE_FEW = 16;             // rows of a workgroup with a wave a row
constexpr int ROUTE_STAGE = ROUTE_ROWS * (ROUTE_COLS + 2);   // rows of 33 words; later 2 words a choice and 2 more of a row

struct RouteArgs {
    const void* logits;
    const uint8_t* mask;
    int rows, experts, k, normalize, blocks;
    float* weights;
    int32_t *chosen, *slots, *offsets, *source;
    int32_t* counts;                                         // the workspace: [blocks, experts], scanned [blocks + 1, experts]
};

// Exclusive scan of `v` over the workgroup's first 512 threads, in `words` (an int of LDS a wave).  `all`: the sum.
__device__ __forceinline__ int exclusive_scan(int v, int* words, int& all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int sum = wave_scan<false>(v);
    if (lane == 63) words[wave] = sum;
    __syncthreads();
    int before = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < ROUTE_WORDS; ++w) {
        if (w < wave) before += words[w];
        all += words[w];
    }
    return before + sum - v;
}

template <typename T, int KM, bool WHOLE>
__global__ __launch_bounds__(2 * ROUTE_ROWS) void expert_choose_kernel(RouteArgs a) {
    constexpr int HALF = ROUTE_COLS / 2;
    __shared__ float stage[ROUTE_STAGE];
    extern __shared__ unsigned long long bits[];                // [experts][ROUTE_WORDS]
    const int tid = threadIdx.x, half = tid / ROUTE_ROWS, t = tid % ROUTE_ROWS, row0 = blockIdx.x * ROUTE_ROWS, row = row0 + t;
    const bool live = row < a.rows && (!a.mask || a.mask[row] != 0);
    for (int i = tid; i < a.experts * ROUTE_WORDS; i += 2 * ROUTE_ROWS) bits[i] = 0;

    float top[KM];
    int best[KM];
#pragma unroll
    for (int i = 0; i < KM; ++i) {
        top[i] = -INFINITY;
        best[i] = -1;
    }
    float sum = 0.f, sum_at = -INFINITY;           // of exp(v - sum_at) over what the thread has seen
    // A thread fetches 8 experts of 2 rows, 4 threads a row; the next experts are on their way while these are walked.  A piece
    // that would end behind the row is moved back to its last 8 experts, so that no load stands in a branch (WHOLE: 8 or more).
    T next[2][8];
    const int piece = (tid & 3) * 8;
    auto fetch = [&](int c0) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int64_t r = min(row0 + (tid >> 2) + i * (ROUTE_ROWS / 2), a.rows - 1);
            const T* p = (const T*)a.logits + r * a.experts;
            if (WHOLE) {
                __builtin_memcpy(next[i], p + min(c0 + piece, a.experts - 8), sizeof(next[i]));
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) next[i][j] = p[min(piece + j, a.experts - 1)];
            }
        }
    };
    fetch(0);
    for (int c0 = 0; c0 < a.experts; c0 += ROUTE_COLS) {
        const int back = WHOLE ? max(0, c0 + piece - (a.experts - 8)) : 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float* to = stage + ((tid >> 2) + i * (ROUTE_ROWS / 2)) * (ROUTE_COLS + 1) + piece;
            if (back == 0) {
#pragma unroll
                for (int j = 0; j < 8; ++j) to[j] = (float)next[i][j];
            } else {
#pragma unroll
                for (int j = 1; j < 8; ++j)
                    if (j >= back) to[j - back] = (float)next[i][j];
            }
        }
        __syncthreads();
        if (c0 + ROUTE_COLS < a.experts) fetch(c0 + ROUTE_COLS);
        const int first = c0 + half * HALF, cols = min(HALF, a.experts - first);
        if (live && cols > 0) {
            const float* mine = stage + t * (ROUTE_COLS + 1) + half * HALF;
#pragma unroll 4
            for (int c = 0; c < cols; ++c) {
                // sorted insert: an entry becomes the middle one of itself, the one above and v; equal values stay in front
                const float v = fmaxf(mine[c], -INFINITY);          // not a number: the smallest
                bool here[KM];
#pragma unroll
                for (int i = 0; i < KM; ++i) here[i] = v > top[i];
#pragma unroll
                for (int i = KM - 1; i > 0; --i) {
                    top[i] = __builtin_amdgcn_fmed3f(top[i - 1], top[i], v);
                    best[i] = here[i - 1] ? best[i - 1] : (here[i] ? first + c : best[i]);
                }
                top[0] = fmaxf(top[0], v);
                best[0] = here[0] ? first + c : best[0];
            }
            if (!a.normalize && top[0] > -INFINITY) {
                if (sum_at != top[0]) sum = sum_at == -INFINITY ? 0.f : sum * exp_fast(sum_at - top[0]);
                sum_at = top[0];
                if (sum_at < INFINITY) {
                    // exp2 without exp_fast's second term: its relative error grows with the distance that makes the value small.
                    // Four sums in turn, so that no value goes through more than a few roundings; a distance that is no number or
                    // too long for anything but zero counts as 200
                    float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
#pragma unroll 4
                    for (int c = 0; c < cols; ++c) {
                        const float next = s0 + __builtin_amdgcn_exp2f(fmaxf(mine[c] - sum_at, -200.f) * 1.44269504088896341f);
                        s0 = s1;
                        s1 = s2;
                        s2 = s3;
                        s3 = next;
                    }
                    sum += (s0 + s1) + (s2 + s3);
                } else {
                    for (int c = 0; c < cols; ++c) sum += mine[c] == INFINITY ? 1.f : 0.f;
                }
            }
        }
    }

    // the second thread's choices and sum go to the first
    __syncthreads();
    float* his = stage + t;
    if (half == 1) {
#pragma unroll
        for (int i = 0; i < KM; ++i) {
            his[2 * i * ROUTE_ROWS] = top[i];
            his[(2 * i + 1) * ROUTE_ROWS] = __int_as_float(best[i]);
        }
        his[2 * KM * ROUTE_ROWS] = sum;
        his[(2 * KM + 1) * ROUTE_ROWS] = sum_at;
    }
    __syncthreads();
    if (half == 0) {
        const float other = his[2 * KM * ROUTE_ROWS], other_at = his[(2 * KM + 1) * ROUTE_ROWS], at = fmaxf(sum_at, other_at);
        if (at > -INFINITY)
            sum = (sum_at == at ? sum : (sum_at == -INFINITY ? 0.f : sum * exp_fast(sum_at - at))) +
                  (other_at == at ? other : (other_at == -INFINITY ? 0.f : other * exp_fast(other_at - at)));
#pragma unroll
        for (int q = 0; q < KM; ++q) {
            const float v = his[2 * q * ROUTE_ROWS];
            const int x = __float_as_int(his[(2 * q + 1) * ROUTE_ROWS]);
            if (x < 0) break;
            bool here[KM];
#pragma unroll
            for (int i = 0; i < KM; ++i) here[i] = v > top[i] || (v == top[i] && x < best[i]);
#pragma unroll
            for (int i = KM - 1; i > 0; --i) {
                top[i] = here[i - 1] ? top[i - 1] : (here[i] ? v : top[i]);
                best[i] = here[i - 1] ? best[i - 1] : (here[i] ? x : best[i]);
            }
            top[0] = here[0] ? v : top[0];
            best[0] = here[0] ? x : best[0];
        }
    } else {
#pragma unroll
        for (int i = 0; i < KM; ++i) best[i] = -1;
    }

    float e[KM];
    float chosen_sum = 0.f;
#pragma unroll
    for (int i = 0; i < KM; ++i) {
        const bool is = i < a.k && best[i] >= 0;
        e[i] = !is ? 0.f : (top[i] == top[0] ? 1.f : expf(top[i] - top[0]));
        chosen_sum += e[i];
        if (is) atomicOr(&bits[best[i] * ROUTE_WORDS + (t >> 6)], 1ull << (t & 63));
    }
    if (a.normalize) sum = chosen_sum;
    __syncthreads();

    // counts of this workgroup; with one workgroup they are the totals
    int n = 0;
    if (t < a.experts)
#pragma unroll
        for (int w = 0; w < ROUTE_WORDS; ++w) n += __popcll(bits[t * ROUTE_WORDS + w]);
    static_assert(2 * FD_ROUTE_MAX_K + 2 <= ROUTE_COLS + 2, "what the second thread hands over fits the stage");
    int* base = (int*)stage;
    if (a.blocks == 1) {
        int all;
        const int first = exclusive_scan(n, base + ROUTE_ROWS, all);
        if (half == 0) {
            base[t] = first;
            if (t < a.experts) a.offsets[t] = first;
            if (t == 0) a.offsets[a.experts] = all;
        }
        __syncthreads();
        for (int i = all + tid; i < a.rows * a.k; i += 2 * ROUTE_ROWS) a.source[i] = -1;
    } else if (half == 0 && t < a.experts) {
        a.counts[(int64_t)blockIdx.x * a.experts + t] = n;
    }
    if (half == 1 || row >= a.rows) return;
#pragma unroll
    for (int i = 0; i < KM; ++i) {
        if (i >= a.k) continue;
        int at = -1;
        if (best[i] >= 0) {
            const unsigned long long* b = bits + best[i] * ROUTE_WORDS;
            at = __popcll(b[t >> 6] & ((1ull << (t & 63)) - 1));
            for (int w = 0; w < (t >> 6); ++w) at += __popcll(b[w]);
            if (a.blocks == 1) {
                at += base[best[i]];
                a.source[at] = row;
            }
        }
        a.weights[(int64_t)row * a.k + i] = best[i] >= 0 ? e[i] / sum : 0.f;
        a.chosen[(int64_t)row * a.k + i] = best[i];
        a.slots[(int64_t)row * a.k + i] = at;                  // several workgroups: the rank, placed below
    }
}

// Largest value of a wave, or its sum, in every lane: shifts within rows of 16 lanes, then row 0 to 1 and 2 to 3, then the half.
template <bool SUM>
__device__ __forceinline__ float wave_all(float v) {
#define FD_STEP(CTRL, ROWS)                                                                                   \
    {                                                                                                         \
        const int bits = __float_as_int(v);                                                                   \
        const float from = __int_as_float(__builtin_amdgcn_update_dpp(SUM ? 0 : bits, bits, CTRL, ROWS, 0xf, false)); \
        v = SUM ? v + from : fmaxf(v, from);                                                                  \
    }
    FD_STEP(0x111, 0xf) FD_STEP(0x112, 0xf) FD_STEP(0x114, 0xf) FD_STEP(0x118, 0xf) FD_STEP(0x142, 0xa) FD_STEP(0x143, 0xc)
#undef FD_STEP
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

// Rows that would not fill the GPU at two threads a row: a wave takes one, experts VALUES * l .. in lane l, and finds its choices
// one by one, ROUTE_FEW rows a workgroup (10 rows of 8 experts, 2 choices: 2.6 us; 16, 32 and 64 rows a workgroup of 16
// waves, one after another or side by side, 4096 rows of 64 experts, 4 choices: 8.7, 9.5 and 13.5 us).
template <typename T, int VALUES, bool MANY>
__global__ __launch_bounds__(64 * ROUTE_FEW) void expert_choose_few_kernel(RouteArgs a) {
    __shared__ unsigned bits[FD_ROUTE_MAX_EXPERTS];          // of an expert: a bit a row
    __shared__ int best[ROUTE_FEW * FD_ROUTE_MAX_K], base[ROUTE_ROWS], words[ROUTE_FEW];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int row0 = MANY ? blockIdx.x * ROUTE_FEW : 0, rows = min(ROUTE_FEW, a.rows - row0), row = row0 + wave;
    for (int i = tid; i < a.experts; i += 64 * ROUTE_FEW) bits[i] = 0;
    __syncthreads();
    if (wave < rows) {
        const bool live = !a.mask || a.mask[row] != 0;
        const T* p = (const T*)a.logits + (int64_t)row * a.experts;
        float v[VALUES];
#pragma unroll
        for (int i = 0; i < VALUES; ++i) {
            const int x = lane * VALUES + i;
            const float l = fmaxf((float)p[min(x, a.experts - 1)], -INFINITY);       // not a number: the smallest
            v[i] = live && x < a.experts ? l : -INFINITY;
        }
        float first = -INFINITY, top = -INFINITY, sum = 0.f;                 // lane j keeps choice j
        int chosen = -1;
        for (int j = 0; j < a.k; ++j) {
            float mine = v[0];
            int x = 0;
#pragma unroll
            for (int i = 1; i < VALUES; ++i) {
                x = v[i] > mine ? i : x;
                mine = fmaxf(mine, v[i]);
            }
            const float most = wave_all<false>(mine);
            if (most == -INFINITY) break;
            if (j == 0) {
                first = most;
                if (!a.normalize)
#pragma unroll
                    for (int i = 0; i < VALUES; ++i) sum += v[i] == most ? 1.f : (v[i] > -INFINITY ? exp_fast(v[i] - most) : 0.f);
            }
            // the lowest expert that has it loses it
            const int src = __ffsll((unsigned long long)__ballot(mine == most)) - 1;
            const int who = __builtin_amdgcn_readlane(lane * VALUES + x, src);
            if (lane == j) {
                top = most;
                chosen = who;
            }
#pragma unroll
            for (int i = 0; i < VALUES; ++i) v[i] = lane == src && x == i ? -INFINITY : v[i];
        }
        const float e = chosen < 0 ? 0.f : (top == first ? 1.f : exp_fast(top - first));
        sum = wave_all<true>(a.normalize ? e : sum);
        if (lane < a.k) {
            const int64_t i = (int64_t)row * a.k + lane;
            a.weights[i] = chosen >= 0 ? e / sum : 0.f;
            a.chosen[i] = chosen;
            best[wave * a.k + lane] = chosen;
            if (chosen >= 0) atomicOr(&bits[chosen], 1u << wave);
        }
    }
    __syncthreads();
    const int n = tid < a.experts ? __popc(bits[tid]) : 0;
    int all = 0;
    if (MANY) {
        if (tid < a.experts) a.counts[(int64_t)blockIdx.x * a.experts + tid] = n;
    } else {
        const int begin = exclusive_scan(n, words, all);
        if (tid < ROUTE_ROWS) {
            base[tid] = begin;
            if (tid < a.experts) a.offsets[tid] = begin;
        }
        if (tid == 0) a.offsets[a.experts] = all;
        __syncthreads();
    }
    for (int i = tid; i < rows * a.k; i += 64 * ROUTE_FEW) {
        const int r = i / a.k, x = best[i];
        int at = -1;
        if (x >= 0) {
            at = __popc(bits[x] & ((1u << r) - 1));
            if (!MANY) {
                at += base[x];
                a.source[at] = r;
            }
        }
        a.slots[(int64_t)row0 * a.k + i] = at;                 // several workgroups: the rank, placed below
        if (!MANY && i >= all) a.source[i] = -1;
    }
}

// The counts of each expert become those of all earlier workgroups, with the sum behind the last.  A workgroup takes 16 experts
// (64-byte pieces of the rows), 64 threads share one.
__global__ __launch_bounds__(1024) void expert_scan_kernel(RouteArgs a) {
    constexpr int PARTS = 64, U = 16;
    __shared__ int sums[PARTS][17];
    const int lane = threadIdx.x & 15, part = threadIdx.x >> 4, e = min((int)blockIdx.x * 16 + lane, a.experts - 1);
    const bool mine = blockIdx.x * 16 + lane < a.experts;
    const int each = (a.blocks + PARTS - 1) / PARTS, b0 = min(part * each, a.blocks), b1 = min(b0 + each, a.blocks);
    int32_t* counts = a.counts + e;
    int n = 0;
#pragma unroll 16
    for (int b = b0; b < b1; ++b) n += counts[(int64_t)b * a.experts];
    sums[part][lane] = n;
    __syncthreads();
    int at = 0;
    for (int p = 0; p < part; ++p) at += sums[p][lane];
    if (!mine) return;
    for (int b = b0; b < b1; b += U) {
        int c[U];
#pragma unroll
        for (int u = 0; u < U; ++u) c[u] = counts[(int64_t)min(b + u, b1 - 1) * a.experts];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (b + u < b1) {
                counts[(int64_t)(b + u) * a.experts] = at;
                at += c[u];
            }
    }
    if (part == PARTS - 1) counts[(int64_t)a.blocks * a.experts] = at;
}

// Adds to every choice's rank the choices of earlier experts and of earlier workgroups (of PER rows).  SUMS: each workgroup sums the
// counts of all.
template <bool SUMS, int PER>
__global__ __launch_bounds__(ROUTE_ROWS) void expert_place_kernel(RouteArgs a) {
    __shared__ int before[ROUTE_ROWS], words[ROUTE_WORDS];
    const int t = threadIdx.x;
    // a thread's first choices are asked for before the counts, whose sums they wait for
    const int64_t i0 = (int64_t)blockIdx.x * PER * a.k, end = min(i0 + PER * a.k, (int64_t)a.rows * a.k);
    int c4[4], r4[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int64_t i = i0 + t + j * ROUTE_ROWS;
        c4[j] = i < end ? a.chosen[i] : -1;
        r4[j] = i < end ? a.slots[i] : -1;
    }
    int b0 = 0, all = 0;
    if (SUMS) {
        // 512 / lanes threads share an expert, each sums every (512 / lanes)-th workgroup
        constexpr int U = 16;
        __shared__ int total[ROUTE_ROWS];
        int lanes = 1;
        while (lanes < a.experts) lanes *= 2;
        const int e = t & (lanes - 1), part = t / lanes, parts = ROUTE_ROWS / lanes;
        if (e < a.experts)
            for (int b = part; b < a.blocks; b += U * parts) {
                int n[U];
#pragma unroll
                for (int u = 0; u < U; ++u) n[u] = a.counts[(int64_t)min(b + u * parts, a.blocks - 1) * a.experts + e];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (b + u * parts < a.blocks) all += n[u];
                    if (b + u * parts < (int)blockIdx.x) b0 += n[u];
                }
            }
        before[t] = b0;
        total[t] = all;
        __syncthreads();
        b0 = all = 0;
        if (t < a.experts)
            for (int p = 0; p < parts; ++p) {
                b0 += before[p * lanes + t];
                all += total[p * lanes + t];
            }
        __syncthreads();
    } else if (t < a.experts) {
        b0 = a.counts[(int64_t)blockIdx.x * a.experts + t];
        all = a.counts[(int64_t)a.blocks * a.experts + t];
    }
    int routed;
    const int first = exclusive_scan(all, words, routed);
    before[t] = first + b0;
    if (blockIdx.x == 0) {
        if (t < a.experts) a.offsets[t] = first;
        if (t == 0) a.offsets[a.experts] = routed;
    }
    __syncthreads();
    auto place = [&](int64_t i, int x, int rank) {
        if (x >= 0) {
            const int at = before[x] + rank;
            a.slots[i] = at;
            a.source[at] = (int)(i / a.k);
        }
        if (i >= routed) a.source[i] = -1;
    };
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (i0 + t + j * ROUTE_ROWS < end) place(i0 + t + j * ROUTE_ROWS, c4[j], r4[j]);
    for (int64_t i = i0 + t + 4 * ROUTE_ROWS; i < end; i += ROUTE_ROWS) place(i, a.chosen[i], a.slots[i]);
}

// Whether the counts of the workgroups are scanned by a launch of their own, which takes some 4 us, rather than summed by every
// workgroup of the next (2048 and 4096 rows of 512 experts, 2 choices, 16 rows a workgroup: 13.9 and 15.1 us with the scan, 16.9
// without it at 2048; 524288 and 1048576 rows of 64, 4 choices: 62 and 112 us, 69 and 147 without).
static bool route_scans(int64_t blocks, int experts) { return blocks > 1024 || blocks * experts > 16384; }

// Rows of a workgroup, which is also the choice of the kernel: a wave a row where that many rows at two threads each leave most
// CUs idle and the experts are enough for 64 lanes (4096 rows: of 16 experts, 8 choices, 9.5 us, walk 19.1; of 64, 4 choices,
// 9.3 and 16.8; of 512, 16 choices, 23 and 169; 16384 rows of 64, 4 choices: 17.1 both; 32768 of 128, 4 choices: 31 and 24).
// Up to 512 rows the walk is a single launch (256 rows: of 8 experts, 2 choices, 7.8 and 5.5 us; of 32, 8 choices, 8.7 and 14).
static int route_rows(int64_t rows, int experts) {
    const int64_t fill = 128 * experts < 32768 ? 128 * experts : 32768;
    const bool few = rows <= ROUTE_FEW || (experts >= (rows <= ROUTE_ROWS ? 32 : 16) && rows <= (fill > 8192 ? fill : 8192));
    return few ? ROUTE_FEW : ROUTE_ROWS;
}

template <typename T>
static void launch_choose(const RouteArgs& a, bool few, hipStream_t s) {
    const dim3 grid(a.blocks), block(2 * ROUTE_ROWS);
    if (few) {
        const dim3 threads(64 * ROUTE_FEW);
#define FD_FEW(VALUES)                                                                                                 \
    do {                                                                                                               \
        if (a.blocks == 1) hipLaunchKernelGGL((expert_choose_few_kernel<T, VALUES, false>), grid, threads, 0, s, a);   \
        else hipLaunchKernelGGL((expert_choose_few_kernel<T, VALUES, true>), grid, threads, 0, s, a);                  \
    } while (0)
        if (a.experts <= 64) FD_FEW(1);
        else if (a.experts <= 256) FD_FEW(4);
        else FD_FEW(8);
#undef FD_FEW
        return;
    }
    const size_t lds = (size_t)a.experts * ROUTE_WORDS * sizeof(unsigned long long);
#define FD_CHOOSE(KM, WHOLE) hipLaunchKernelGGL((expert_choose_kernel<T, KM, WHOLE>), grid, block, lds, s, a)
    if (a.experts < 8) {
        if (a.k <= 2) FD_CHOOSE(2, false);
        else FD_CHOOSE(8, false);
    } else if (a.k == 1) FD_CHOOSE(1, true);
    else if (a.k == 2) FD_CHOOSE(2, true);
    else if (a.k <= 4) FD_CHOOSE(4, true);
    else if (a.k <= 8) FD_CHOOSE(8, true);
    else FD_CHOOSE(16, true);
#undef FD_CHOOSE
}

static void launch_place(const RouteArgs& a, bool few, hipStream_t s) {
    const dim3 grid(a.blocks), block(ROUTE_ROWS);
    if (!route_scans(a.blocks, a.experts)) {
        if (few) hipLaunchKernelGGL((expert_place_kernel<true, ROUTE_FEW>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((expert_place_kernel<true, ROUTE_ROWS>), grid, block, 0, s, a);
    } else {
        if (few) hipLaunchKernelGGL((expert_place_kernel<false, ROUTE_FEW>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((expert_place_kernel<false, ROUTE_ROWS>), grid, block, 0, s, a);
    }
}

}  // namespace fd

extern "C" {

int64_t fd_expert_route_workspace(int64_t rows, int experts) {
    const int per = fd::route_rows(rows, experts);
    const int64_t blocks = (rows + per - 1) / per;
    return blocks > 1 ? (blocks + fd::route_scans(blocks, experts)) * experts * (int64_t)sizeof(int32_t) : 0;
}

int fd_expert_route(const void* logits, int dtype, int64_t rows, int experts, int k, const uint8_t* mask, int normalize, float* weights,
                    int32_t* chosen, int32_t* slots, int32_t* offsets, int32_t* source_rows, void* workspace, int64_t workspace_bytes,
                    void* stream) {
    FD_REQUIRE(fd::valid_dtype(dtype), "fd_expert_route: unknown element type");
    FD_REQUIRE(rows >= 0 && experts > 0 && k > 0 && k <= experts, "fd_expert_route: bad shape (rows %lld, experts %d, k %d)", (long long)rows,
               experts, k);
    if (experts > FD_ROUTE_MAX_EXPERTS || k > FD_ROUTE_MAX_K || rows * k >= (int64_t(1) << 31) - 1024) {
        fd::set_error("fd_expert_route: at most %d experts, %d choices a row and 2^31 - 1024 choices", FD_ROUTE_MAX_EXPERTS, FD_ROUTE_MAX_K);
        return FD_ERR_LIMIT;
    }
    FD_REQUIRE(offsets && (rows == 0 || (logits && weights && chosen && slots && source_rows)), "fd_expert_route: NULL pointer");
    FD_REQUIRE(workspace_bytes >= fd_expert_route_workspace(rows, experts) && (workspace || workspace_bytes <= 0),
               "fd_expert_route: a workspace of %lld bytes is needed", (long long)fd_expert_route_workspace(rows, experts));
    fd::RouteArgs a;
    a.logits = logits; a.mask = mask; a.rows = (int)rows; a.experts = experts; a.k = k; a.normalize = normalize != 0;
    const int per = fd::route_rows(rows, experts);
    a.blocks = rows ? fd::ceil_div(rows, per) : 1;
    a.weights = weights; a.chosen = chosen; a.slots = slots; a.offsets = offsets; a.source = source_rows; a.counts = (int32_t*)workspace;
    fd::ProfScope scope(fd::as_stream(stream), "expert_route", (double)rows * experts * (2 + k),
                        (double)rows * experts * fd::dtype_bytes(dtype) + 16.0 * rows * k);
    return fd::with_dtype(dtype, [&](auto t) {
        fd::launch_choose<decltype(t)>(a, per == fd::ROUTE_FEW, fd::as_stream(stream));
        FD_LAUNCH_CHECK();
        if (a.blocks > 1) {
            if (fd::route_scans(a.blocks, experts)) {
                hipLaunchKernelGGL(fd::expert_scan_kernel, dim3(fd::ceil_div(experts, 16)), dim3(1024), 0, fd::as_stream(stream), a);
                FD_LAUNCH_CHECK();
            }
            fd::launch_place(a, per == fd::ROUTE_FEW, fd::as_stream(stream));
            FD_LAUNCH_CHECK();
        }
        return FD_OK;
    });
}

}  // extern "C"
