// Attention of packed prompts with grouped heads, a sliding window and sinks, sm_100a:
//
//   o[i, h, :] = sum_j softmax_j(scale q[i, h, :] . k[j, h / g, :]) v[j, h / g, :]
//   query i of a sequence with nq queries and nk keys sits at position p = i + nk - nq and sees the
//   keys j <= p with j > p - window or j < sinks (window 0: all j <= p)
//
// q, o [Tq, Hq, D] and k, v [Tk, Hk, D] with any token and head strides, g = Hq / Hk, sequences packed
// by cu_seqlens; fp16 / bf16, softmax statistics in fp32.  A query that sees nothing gives zeros; rows
// of no sequence are left as they were.
#include "sf_common.cuh"
#include "sm100.cuh"
#include "tma_host.cuh"

#include <algorithm>
#include <cmath>

namespace {

constexpr float LOG2E = 1.4426950408889634f;

struct Args {
    const void *q, *k, *v;
    void* o;
    const int32_t *cu_q, *cu_k;
    int64_t qt, qh, kt, kh, vt, vh, ot, oh;  // strides in elements
    int64_t tq, tk;
    int seqs, group, heads;                  // sequences, query heads a kv head, query heads
    int window, sinks;
    float scale_log2;
};

// Keys [0, sinks) and [low, high) of a query at position p.
struct Keys {
    int sinks, low, high;
    __device__ __forceinline__ Keys(const Args& a, int p) {
        high = max(0, p + 1);
        low = a.window ? max(0, p - a.window + 1) : 0;
        sinks = min(a.sinks, low);
    }
};

// A sequence's first and end row, inside [0, total) whatever the table holds.
__device__ __forceinline__ void bounds(const int32_t* cu, int s, int64_t total, int64_t* begin, int64_t* end) {
    *begin = min((int64_t)max(0, __ldg(cu + s)), total);
    *end = max(*begin, min((int64_t)max(0, __ldg(cu + s + 1)), total));
}

// One query row by one warp in fp32, key after key: lane owns elements lane + 32 e (D <= 256).
template <typename T>
__device__ __forceinline__ void row_by_warp(const Args& a, int D, int64_t qrow, int head, int64_t kbegin, int p, T* out) {
    const int lane = threadIdx.x & 31;
    const T* q = (const T*)a.q + qrow * a.qt + (int64_t)head * a.qh;
    const T* k = (const T*)a.k + kbegin * a.kt + (int64_t)(head / a.group) * a.kh;
    const T* v = (const T*)a.v + kbegin * a.vt + (int64_t)(head / a.group) * a.vh;
    float qv[8], acc[8], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        qv[e] = lane + 32 * e < D ? sf::Dt<T>::to_f(q[lane + 32 * e]) : 0.f;
        acc[e] = 0.f;
    }
    const Keys keys(a, p);
    const int n = keys.sinks + keys.high - keys.low;
    for (int i = 0; i < n; ++i) {
        const int64_t j = i < keys.sinks ? i : keys.low + (i - keys.sinks);
        float dot = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (lane + 32 * e < D) dot = fmaf(qv[e], sf::Dt<T>::to_f(k[j * a.kt + lane + 32 * e]), dot);
        const float s = sf::warp_sum(dot) * a.scale_log2;
        const float mx = s > m || s != s ? s : m;
        const float shift = mx == -INFINITY ? 0.f : mx;
        const float f = exp2f(m - shift), w = exp2f(s - shift);
        l = l * f + w;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (lane + 32 * e < D) acc[e] = acc[e] * f + w * sf::Dt<T>::to_f(v[j * a.vt + lane + 32 * e]);
        m = mx;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (lane + 32 * e < D) out[lane + 32 * e] = sf::Dt<T>::from_f(n ? acc[e] / l : 0.f);
}

// ---- general kernel: a warp a (query, head) row, any D <= 256, strides and alignment -------------
template <typename T>
__global__ void __launch_bounds__(128) window_general_kernel(const Args a, int D) {
    const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (i >= a.tq * a.heads) return;
    const int64_t row = i / a.heads;
    const int head = (int)(i - row * a.heads);
    int lo = 0, hi = a.seqs;  // the last sequence that begins at or before the row
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (__ldg(a.cu_q + mid) <= row) lo = mid;
        else hi = mid;
    }
    int64_t qb, qe, kb, ke;
    bounds(a.cu_q, lo, a.tq, &qb, &qe);
    bounds(a.cu_k, lo, a.tk, &kb, &ke);
    if (row < qb || row >= qe) return;
    const int p = (int)((row - qb) + (ke - kb) - (qe - qb));
    row_by_warp<T>(a, D, row, head, kb, p, (T*)a.o + row * a.ot + (int64_t)head * a.oh);
}

template <typename T>
int launch_general(const Args& a, int64_t D, cudaStream_t st, char* err, uint64_t cap) {
    if (D > 256) return sf::fail(SF_EINVAL, err, cap, "window_attention: D=%lld exceeds 256", (long long)D);
    const int64_t blocks = (a.tq * a.heads + 3) / 4;
    if (blocks > 0x7fffffffLL) return sf::fail(SF_EINVAL, err, cap, "window_attention: grid too large");
    window_general_kernel<T><<<(unsigned)blocks, 128, 0, st>>>(a, (int)D);
    return sf::check_launch("window_attention general launch", err, cap);
}

}  // namespace

int sf_window_attention_launch(const void* q, const void* k, const void* v, const void* cu_q, const void* cu_k, void* o, int64_t Tq, int64_t Tk,
                               int64_t seqs, int64_t Hq, int64_t Hk, int64_t D, const int64_t* strides, float scale, int64_t window, int64_t sinks,
                               int32_t dtype, int32_t variant, cudaStream_t st, char* err, uint64_t cap) {
    if (Tq < 0 || Tk < 0 || seqs < 0 || Hq < 0 || Hk < 0 || D < 1) return sf::fail(SF_EINVAL, err, cap, "window_attention: bad sizes");
    if (Hq && (Hk == 0 || Hq % Hk)) return sf::fail(SF_EINVAL, err, cap, "window_attention: the query heads must be a multiple of the key heads");
    if (Tq > 0x7fffffffLL || Tk > 0x7fffffffLL || seqs > 0x7fffffffLL || Hq > (1 << 20)) return sf::fail(SF_EINVAL, err, cap, "window_attention: size above 2^31 - 1");
    if (!(scale > 0.f) || !(scale < INFINITY)) return sf::fail(SF_EINVAL, err, cap, "window_attention: scale must be > 0");
    if (window < 0 || sinks < 0) return sf::fail(SF_EINVAL, err, cap, "window_attention: window and sinks must be >= 0");
    if (dtype != SF_DTYPE_F16 && dtype != SF_DTYPE_BF16) return sf::fail(SF_EINVAL, err, cap, "window_attention: dtype %d is not fp16/bf16", dtype);
    if (Tq * Hq == 0 || seqs == 0) return SF_OK;
    if (!q || !o || !cu_q || !cu_k || (Tk && (!k || !v))) return sf::fail(SF_EINVAL, err, cap, "window_attention: null tensor pointer");
    const int64_t dense[8] = {Hq * D, D, Hk * D, D, Hk * D, D, Hq * D, D};
    const int64_t* s = strides ? strides : dense;
    for (int i = 0; i < 8; ++i)
        if (s[i] < 0) return sf::fail(SF_EINVAL, err, cap, "window_attention: negative stride");
    Args a = {};
    a.q = q, a.k = k, a.v = v, a.o = o;
    a.cu_q = (const int32_t*)cu_q, a.cu_k = (const int32_t*)cu_k;
    a.qt = s[0], a.qh = s[1], a.kt = s[2], a.kh = s[3], a.vt = s[4], a.vh = s[5], a.ot = s[6], a.oh = s[7];
    a.tq = Tq, a.tk = Tk;
    a.seqs = (int)seqs, a.group = (int)(Hq / Hk), a.heads = (int)Hq;
    a.window = (int)std::min<int64_t>(window, 0x7fffffff);
    a.sinks = window ? (int)std::min<int64_t>(sinks, 0x7fffffff) : 0;
    a.scale_log2 = scale * LOG2E;
    if (variant == 1) return sf::fail(SF_EINVAL, err, cap, "window_attention: no tensor-core kernel yet");
    if (dtype == SF_DTYPE_F16) return launch_general<__half>(a, D, st, err, cap);
    return launch_general<__nv_bfloat16>(a, D, st, err, cap);
}

extern "C" int sf_window_attention(const void* q, const void* k, const void* v, const void* cu_q, const void* cu_k, void* o, int64_t Tq, int64_t Tk,
                                   int64_t seqs, int64_t Hq, int64_t Hk, int64_t D, const int64_t* strides, float scale, int64_t window,
                                   int64_t sinks, int32_t dtype, int32_t variant, void* stream, char* err, uint64_t cap) {
    return sf_window_attention_launch(q, k, v, cu_q, cu_k, o, Tq, Tk, seqs, Hq, Hk, D, strides, scale, window, sinks, dtype, variant, (cudaStream_t)stream,
                                      err, cap);
}
