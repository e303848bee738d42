// The router's balance loss: counts of the selections, mean softmax probabilities, their product, and its gradient.
//
//   loss = coef * E / (N k) * sum_e counts[e] * P[e],   P[e] = 1/N * sum over the counted tokens t of p[t][e],   p = softmax over the E logits
//   d loss / d logit[t][j] = p[t][j] * (g[j] - sum_e p[t][e] g[e]),   g[e] = d_loss * coef * E / (N^2 k) * counts[e]
//
// N: tokens that the mask leaves.  The counts have no gradient.  A logit that is not finite is taken as -3.4e38, as the selection takes it
// (shaders/moe_select.comp:28-34), and gets none.  A warp holds a row in registers, the same columns in the same lane for every row, so a lane adds up its
// columns' probabilities - and keeps its columns' g - in registers.
//
// What bounds it at 32768 x 256: the loss (14.9 us; 33.5 MB, 5.1 at the copy rate) issues some 25 instructions an element, and ends with additions of all blocks to
// the same sums and a kernel that reads them; the gradient (14.4 us; 67 MB, 10.2) is near its traffic.
#include <cmath>
#include <type_traits>

#include "qkm_common.cuh"
#include "qkm_kernels.h"

namespace qkm {
namespace {

constexpr int kBalThreads = 256, kBalWarps = kBalThreads / 32;
constexpr float kFloor = -3.4e38f;
// Sums over blocks are added as integers of 1 / fix: whatever their order, the result is the same.  A sum is n_tokens at most, so fix is 2^62 over the power
// of two that n_tokens does not pass: the sums stay inside 64 bits, and a mean is off by 2^-63 of that power at most (a rounding for each block that has a token
// which counts): less than f32 rounds down to probabilities of 2^-39 where there is one token (2^-38 as fixed a unit lost those below 2^-15).
double bal_fix(uint32_t n_tokens) {
    int up = 0;
    while (n_tokens > 1u << up) ++up;
    return ldexp(1.0, 62 - up);
}

// Sums of balance_kernel, which balance_finish_kernel reads and sets back to zero.  Calls of two streams that overlap add to the same sums and get wrong
// results; but whichever of their finish kernels runs last has every addition before it and leaves zeros, so that nothing of them reaches a later call.
// (With the last block of one kernel, told by a count, in place of the second kernel, the count and the sums could stay wrong for good.)
struct BalanceAcc {
    unsigned long long p[512];
    uint32_t counts[512];
    uint32_t kept;
};

// V values a lane: column of value i
template <bool VEC> __device__ __forceinline__ uint32_t bal_col(uint32_t lane, int i) { return VEC ? ((i >> 2) * 32 + lane) * 4 + (i & 3) : i * 32 + lane; }

// rows that a warp has under way at once (32768 x 256: two 14.9 + 14.7 us, four 15.9 + 17.7; 32768 x 128: 13.0 + 12.8 against 11.9 + 11.5)
template <int V> constexpr int bal_rows() { return V <= 4 ? 4 : 2; }

constexpr float kLowest = -3.402823466e38f;   // stands for a logit past the end of a row, below any that counts

template <int V, bool VEC>
__device__ __forceinline__ void row_load(const float* row, uint32_t E, uint32_t lane, float (&v)[V]) {
    if (VEC) {
#pragma unroll
        for (int j = 0; j < V / 4; ++j) {
            const uint32_t c = bal_col<VEC>(lane, 4 * j);
            float4 f = make_float4(kLowest, kLowest, kLowest, kLowest);
            if (c < E) f = *reinterpret_cast<const float4*>(row + c);
            v[4 * j] = f.x; v[4 * j + 1] = f.y; v[4 * j + 2] = f.z; v[4 * j + 3] = f.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = bal_col<VEC>(lane, i) < E ? row[bal_col<VEC>(lane, i)] : kLowest;
    }
}
__device__ __forceinline__ float warp_max(float v) {
    float r;
    asm("redux.sync.max.f32 %0, %1, 0xFFFFFFFF;" : "=f"(r) : "f"(v));
    return r;
}
// e^x for x <= 0, to about 3 * 2^-24 of it, 0 below 2^-126: 2^t for t = x log2(e) rounded, times 1 + ln 2 times what the rounding of the product
// (r, which an FMA gives exactly) and of log2(e) left out.
__device__ __forceinline__ float exp_down(float x) {
    constexpr float kLog2e = 1.44269504f, kRest = 1.92596303e-8f, kLn2 = 0.693147181f;   // log2(e) = kLog2e + kRest
    x = fmaxf(x, -1e4f);                       // (0 from -88 on, and t stays finite)
    const float t = x * kLog2e, r = fmaf(x, kLog2e, -t), c = fmaf(x, kRest * kLn2, r * kLn2);
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
    return fmaf(e, c, e);
}
// A row's logits -> exp(logit - largest), 0 past the end; returns 1 / their sum.  Where the largest is above the floor, what is at the floor, or past
// the end, gives 0 by itself; `low` says that it is not, and the caller looks at every element then.
template <int V, bool VEC>
__device__ __forceinline__ float row_exp(uint32_t E, uint32_t lane, float (&v)[V], bool& low) {
    float most = kLowest;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        if (!(fabsf(v[i]) <= -kLowest)) v[i] = kFloor;
        most = fmaxf(most, v[i]);
    }
    most = warp_max(most);
    low = most <= kFloor;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        v[i] = exp_down(v[i] - most);
        if (low && bal_col<VEC>(lane, i) >= E) v[i] = 0.f;
        sum += v[i];
    }
    return __fdividef(1.f, warp_sum(sum));     // (1 <= sum <= 512)
}

// (8 values a lane: without the number of blocks (0: none given) the compiler takes 48 registers and one row's loads at a time, 16.8 us of 32768 x 256 instead of 14.9)
template <int V, bool VEC>
__global__ void __launch_bounds__(kBalThreads, V == 8 ? 4 : 0)
balance_kernel(const float* __restrict__ logits, const qkm_sel* __restrict__ sel, const uint8_t* __restrict__ mask, uint32_t n_tokens, uint32_t E, uint32_t n_used, double fix,
               BalanceAcc* acc) {
    __shared__ float s_p[kBalWarps][V * 32];
    __shared__ uint32_t s_cnt[V * 32];
    __shared__ uint32_t s_kept;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    for (uint32_t i = tid; i < V * 32; i += kBalThreads) s_cnt[i] = 0;
    if (tid == 0) s_kept = 0;
    pdl_trigger();
    pdl_wait();
    __syncthreads();
    float p[V] = {};
    uint32_t kept = 0;
    constexpr int R = bal_rows<V>();
    const uint32_t step = gridDim.x * kBalWarps;
    for (uint32_t t0 = blockIdx.x * kBalWarps + warp; t0 < n_tokens; t0 += R * step) {
        float v[R][V];
        uint32_t id[R];
        bool in[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const uint32_t t = t0 + r * step;      // (below 2^24 + 2^14)
            in[r] = t < n_tokens && !(mask && mask[t] == 0);
            id[r] = 0xFFFFFFFFu;
            if (in[r]) {
                row_load<V, VEC>(logits + (size_t)t * E, E, lane, v[r]);
                if (lane < n_used) id[r] = sel[t].ids[lane];
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (in[r]) {                           // (the same for the whole warp)
                bool low;
                const float inv = row_exp<V, VEC>(E, lane, v[r], low);
#pragma unroll
                for (int i = 0; i < V; ++i) p[i] += v[r][i] * inv;
                if (id[r] < E) atomicAdd(&s_cnt[id[r]], 1u);
                ++kept;
            }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) s_p[warp][bal_col<VEC>(lane, i)] = p[i];
    if (lane == 0 && kept) atomicAdd(&s_kept, kept);
    __syncthreads();
    for (uint32_t e = tid; e < E; e += kBalThreads) {
        double s = 0;
        for (int w = 0; w < kBalWarps; ++w) s += (double)s_p[w][e];
        if (s != 0) atomicAdd(&acc->p[e], (unsigned long long)__double2ll_rn(s * fix));
        if (s_cnt[e]) atomicAdd(&acc->counts[e], s_cnt[e]);
    }
    if (tid == 0 && s_kept) atomicAdd(&acc->kept, s_kept);
}

// One block, a thread an expert; unit: 1 / fix, factor: coef * E / n_used
constexpr int kFinThreads = 512;
__global__ void __launch_bounds__(kFinThreads)
balance_finish_kernel(BalanceAcc* acc, uint32_t E, double unit, double factor, uint32_t* __restrict__ counts, float* __restrict__ probs, float* __restrict__ loss) {
    __shared__ double s_sum[kFinThreads / 32];
    const uint32_t e = threadIdx.x;
    pdl_trigger();
    pdl_wait();
    const uint32_t N = acc->kept;
    const double per = N ? 1.0 / N : 0.0;
    double sum = 0;
    if (e < E) {
        const uint32_t c = acc->counts[e];
        const double P = (double)acc->p[e] * unit * per;
        acc->p[e] = 0; acc->counts[e] = 0;
        counts[e] = c;
        probs[e] = (float)P;
        sum = (double)c * P;
    }
    sum = warp_sum(sum);
    if ((e & 31u) == 0) s_sum[e >> 5] = sum;
    __syncthreads();
    if (e >= 32) return;
    sum = warp_sum(e < kFinThreads / 32 ? s_sum[e] : 0.0);
    if (e == 0) {
        counts[E] = N;
        *loss = (float)(sum * per * factor);
        acc->kept = 0;
    }
}

template <int V>
__device__ __forceinline__ void drop(float (&v)[V], int at) {
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (i == at) v[i] = 0.f;
}

template <int V, bool VEC>
__global__ void __launch_bounds__(kBalThreads)
balance_grad_kernel(const float* logits, const uint8_t* __restrict__ mask, const uint32_t* __restrict__ counts, uint32_t n_tokens, uint32_t E, double factor,
                    const float* __restrict__ d_loss, float* d_logits) {
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    pdl_trigger();
    pdl_wait();
    const uint32_t N = counts[E];
    const double up = d_loss ? (double)*d_loss : 1.0, unit = N ? factor / ((double)N * N) * up : 0.0;
    float g[V];
#pragma unroll
    for (int i = 0; i < V; ++i) g[i] = bal_col<VEC>(lane, i) < E ? (float)(unit * counts[bal_col<VEC>(lane, i)]) : 0.f;
    constexpr int R = bal_rows<V>();
    const uint32_t step = gridDim.x * kBalWarps;
    for (uint32_t t0 = blockIdx.x * kBalWarps + warp; t0 < n_tokens; t0 += R * step) {
        float v[R][V];
        bool in[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const uint32_t t = t0 + r * step;
            in[r] = t < n_tokens && !(mask && mask[t] == 0);
            if (in[r]) row_load<V, VEC>(logits + (size_t)t * E, E, lane, v[r]);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const uint32_t t = t0 + r * step;
            if (t >= n_tokens) break;
            if (in[r]) {
                bool low;
                const float inv = row_exp<V, VEC>(E, lane, v[r], low);
                float dot = 0.f;
#pragma unroll
                for (int i = 0; i < V; ++i) { v[r][i] *= inv; dot += v[r][i] * g[i]; }
                dot = warp_sum(dot);
#pragma unroll
                for (int i = 0; i < V; ++i) v[r][i] *= g[i] - dot;
                // Logits that are not finite get no gradient.  Where every logit is at the floor they count; where some g is not finite (then the row's mean is not
                // either) their zero probability does not make them zero.
                if (low || !isfinite(dot))
#pragma unroll 1
                    for (int i = 0; i < V; ++i)
                        if (bal_col<VEC>(lane, i) < E && !isfinite(logits[(size_t)t * E + bal_col<VEC>(lane, i)])) drop(v[r], i);
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) v[r][i] = 0.f;
            }
            float* out = d_logits + (size_t)t * E;
            if (VEC) {
#pragma unroll
                for (int j = 0; j < V / 4; ++j)
                    if (bal_col<VEC>(lane, 4 * j) < E)
                        *reinterpret_cast<float4*>(out + bal_col<VEC>(lane, 4 * j)) = make_float4(v[r][4 * j], v[r][4 * j + 1], v[r][4 * j + 2], v[r][4 * j + 3]);
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (bal_col<VEC>(lane, i) < E) out[bal_col<VEC>(lane, i)] = v[r][i];
            }
        }
    }
}

// f<V, VEC>() for rows of E logits: 4, 8 or 16 values a lane; 16-byte loads where every row starts on 16 bytes
template <class F>
cudaError_t bal_variant(uint32_t E, bool vec, F f) {
    if (E <= 128) return vec ? f(std::integral_constant<int, 4>{}, std::true_type{}) : f(std::integral_constant<int, 4>{}, std::false_type{});
    if (E <= 256) return vec ? f(std::integral_constant<int, 8>{}, std::true_type{}) : f(std::integral_constant<int, 8>{}, std::false_type{});
    return vec ? f(std::integral_constant<int, 16>{}, std::true_type{}) : f(std::integral_constant<int, 16>{}, std::false_type{});
}
// Blocks: as many as the SMs hold, or fewer where that gives every warp the same number of rounds.
uint32_t bal_grid(uint32_t n_tokens, uint32_t n_sms, uint32_t per_sm, uint32_t rows) {
    const uint32_t most = n_sms * per_sm, want = (n_tokens + kBalWarps - 1) / kBalWarps;
    if (want <= most) return want < 1 ? 1u : want;
    const uint32_t round = most * kBalWarps * rows, rounds = (n_tokens + round - 1) / round;
    return (n_tokens + rounds * rows * kBalWarps - 1) / (rounds * rows * kBalWarps);
}

}  // namespace

size_t balance_scratch_bytes() { return sizeof(BalanceAcc); }

cudaError_t launch_balance(const Launch& L, const qkm_dims& d, const float* logits, const qkm_sel* sel, const uint8_t* mask, uint32_t n_tokens, float coef, void* scratch,
                           uint32_t* counts, float* probs, float* loss, uint32_t n_sms) {
    const Launch P{L.stream, nullptr, true};
    const double fix = bal_fix(n_tokens);
    cudaError_t e = cudaSuccess;
    if (n_tokens) {
        e = bal_variant(d.n_expert, d.n_expert % 4 == 0 && ((uintptr_t)logits & 15u) == 0, [&](auto v, auto vec) {
            return launch_kernel(P, balance_kernel<v.value, vec.value>, dim3(bal_grid(n_tokens, n_sms, v.value <= 8 ? 4 : 3, bal_rows<v.value>())), dim3(kBalThreads), 0, logits, sel, mask,
                                 n_tokens, d.n_expert, d.n_used, fix, (BalanceAcc*)scratch);
        });
        L.count();
        if (e != cudaSuccess) return e;
    }
    e = launch_kernel(P, balance_finish_kernel, dim3(1), dim3(kFinThreads), 0, (BalanceAcc*)scratch, d.n_expert, 1.0 / fix, (double)coef * d.n_expert / d.n_used, counts, probs, loss);
    L.count();
    return e != cudaSuccess ? e : cudaGetLastError();
}

cudaError_t launch_balance_grad(const Launch& L, const qkm_dims& d, const float* logits, const uint8_t* mask, const uint32_t* counts, uint32_t n_tokens, float coef,
                                const float* d_loss, float* d_logits, uint32_t n_sms) {
    if (n_tokens == 0) return cudaSuccess;
    const bool vec = d.n_expert % 4 == 0 && (((uintptr_t)logits | (uintptr_t)d_logits) & 15u) == 0;
    const cudaError_t e = bal_variant(d.n_expert, vec, [&](auto v, auto ve) {
        return launch_kernel(Launch{L.stream, nullptr, true}, balance_grad_kernel<v.value, ve.value>, dim3(bal_grid(n_tokens, n_sms, v.value == 8 ? 6 : 4, bal_rows<v.value>())), dim3(kBalThreads), 0, logits, mask,
                             counts, n_tokens, d.n_expert, (double)coef * d.n_expert / d.n_used, d_loss, d_logits);
    });
    L.count();
    return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace qkm
