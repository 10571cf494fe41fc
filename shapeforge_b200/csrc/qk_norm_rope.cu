// Per-head RMS norm of queries and keys with the rotary embedding in the same pass, sm_100a:
//
//   y = x * rsqrt(mean(x^2) + eps) * w                        over one head's D elements
//   angle_i = position[t] * base^(-i / r),  r = rotary / 2,  i < r
//   out_i     = y_i cos(angle_i) - y_{i+r} sin(angle_i)
//   out_{i+r} = y_i sin(angle_i) + y_{i+r} cos(angle_i)        the other D - 2r elements: out = y
//
// q [T, Hq, D] and k [T, Hk, D] with any token and head strides (views of a packed projection),
// w_q, w_k [D], position [T] int32, fp16 / bf16 in and out, fp32 arithmetic, one rounding.  The
// outputs may be the inputs' own buffers: the lanes that write a row have read all of it.
//
// HBM-bound: T (Hq + Hk) D elements in and out, each moved once.  16384 tokens of 32 + 8 heads of 128 in bf16:
// 57 us, 5.9 TB/s (90 % of a copy); 64 tokens: 3.4 us, the launch and one round of loads.
//  * A row of D elements is held by D/16 lanes, two 8-element chunks a lane; a lane's chunks are c
//    and c + r/8, so both members of a rotated pair sit in one lane and only the sum of squares
//    crosses lanes (2-4 shuffles).
//  * The angle depends on (t, i) alone, so a warp stays with one token, takes sine and cosine of
//    its 8 angles a lane once, and walks the token's heads, two row groups at work and the next four in
//    flight, the next token's among them (asynchronous copies into the lane's own places).  Tokens are
//    split over heads only when there are too few of them to fill the GPU.
//  * The angle is reduced in double precision (a position near 2^20 times a frequency leaves no
//    fraction bits in fp32), in turns: frac(position * base^(-i/r) / 2 pi), |.| <= 1/2, then the
//    special-function sine and cosine of at most pi (absolute error ~2^-21, far below half a step
//    of a 16-bit output).
#include "sf_common.cuh"
#include "sm100.cuh"

#include <cmath>
#include <initializer_list>

namespace {

struct Side {
    const void* x;
    void* y;
    const void* w;
    int64_t xt, xh, yt, yh;  // token and head strides in elements
};

// Sine and cosine of 2 pi * turns.
__device__ __forceinline__ void sincos_turns(double turns, float* s, float* c) {
    const float f = (float)(turns - rint(turns));
    __sincosf(f * 6.283185307f, s, c);
}

template <typename T>
__device__ __forceinline__ void unpack8(const uint4& u, float2 (&v)[4]) {
    v[0] = sf::Pair<T>::to_f2(u.x);
    v[1] = sf::Pair<T>::to_f2(u.y);
    v[2] = sf::Pair<T>::to_f2(u.z);
    v[3] = sf::Pair<T>::to_f2(u.w);
}

template <typename T>
__device__ __forceinline__ uint4 pack8(const float2 (&v)[4]) {
    return make_uint4(sf::Pair<T>::from_f2(v[0]), sf::Pair<T>::from_f2(v[1]), sf::Pair<T>::from_f2(v[2]), sf::Pair<T>::from_f2(v[3]));
}

// 16384 tokens of 40 heads of 128: 4 CTAs of 4 warps an SM 57 us, 3 58.7, 5 61.3, 6 60.7; 4 pairs of groups in the ring
// 57.7; the next groups in registers instead (2 CTAs of 8 warps) 65.
constexpr int WARPS = 4;  // a CTA
constexpr int CTAS = 4;   // an SM
constexpr int AHEAD = 3;  // pairs of row groups in a warp's ring

// LPR lanes a row (a power of two >= D / 16); `items` = tokens x head parts, one warp an item.
template <typename T, int LPR>
__global__ void __launch_bounds__(32 * WARPS, CTAS) qk_norm_rope_kernel(const Side q, const Side k, const int32_t* __restrict__ position, int64_t tokens,
                                                                     int hq, int hk, int D, int r, double ratio, float eps, int parts) {
    constexpr int RPW = 32 / LPR;  // rows a warp holds at once
    // Both weights, in the lanes' order: 16 bytes a chunk (in registers they would cost a third of the warps).
    __shared__ uint4 w_s[2][2][32];
    // The rows in flight: a lane copies its own two chunks of each of a pair's groups and reads them back itself.
    __shared__ uint4 ring_s[WARPS][AHEAD][2][2][32];
    const int lane = threadIdx.x & 31;
    const int p = lane % LPR, sub = lane / LPR;
    const bool live = p < D / 16;
    const bool turned = p < r / 8;
    // Element offsets of the lane's chunks.
    const int e0 = turned ? 8 * p : 2 * r + 16 * (p - r / 8);
    const int e1 = turned ? e0 + r : e0 + 8;
    if (threadIdx.x < LPR && live) {
        if (hq) {
            w_s[0][0][p] = *reinterpret_cast<const uint4*>((const T*)q.w + e0);
            w_s[0][1][p] = *reinterpret_cast<const uint4*>((const T*)q.w + e1);
        }
        if (hk) {
            w_s[1][0][p] = *reinterpret_cast<const uint4*>((const T*)k.w + e0);
            w_s[1][1][p] = *reinterpret_cast<const uint4*>((const T*)k.w + e1);
        }
    }
    // base^(-i/r) / 2 pi of the lane's 8 angles: the first by repeated squaring, then by `ratio`.
    double turn0 = 0.15915494309189533577;
    if (turned) {
        double sq = ratio;
        for (int e = 8 * p; e > 0; e >>= 1) {
            if (e & 1) turn0 *= sq;
            sq *= sq;
        }
    }
    __syncthreads();
    const float inv_d = 1.0f / (float)D;
    const int rows = hq + hk;
    const int groups = (rows + RPW - 1) / RPW;
    const int per = (groups + parts - 1) / parts;
    const int64_t items = tokens * parts;
    const int64_t step = (int64_t)gridDim.x * (blockDim.x >> 5);
    const int64_t first = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    uint4(*ring)[2][2][32] = ring_s[threadIdx.x >> 5];
    // A place in the warp's rows, two groups at a time: token, next group, end of the item's groups.
    struct Cursor {
        int64_t item, t;
        int g, g1;
    };
    auto enter = [&](Cursor& c) {
        c.t = parts == 1 ? c.item : (int64_t)((uint32_t)c.item / (uint32_t)parts);  // items are few when tokens are split
        c.g = (int)(c.item - c.t * parts) * per;
        c.g1 = min(groups, c.g + per);
    };
    auto next = [&](Cursor& c) {
        c.g += 2;
        if (c.g >= c.g1) {
            c.item += step;
            if (c.item < items) enter(c);
        }
    };
    auto row_of = [&](const Cursor& c, int u) {
        const int row = (c.g + u) * RPW + sub;
        return live && c.g + u < c.g1 && row < rows ? row : -1;
    };
    Cursor ahead = {first, 0, 0, 0};
    if (first < items) enter(ahead);
    Cursor at = ahead;
    auto fetch = [&](int stage) {
        if (ahead.item < items) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int row = row_of(ahead, u);
                if (row >= 0) {
                    const T* x = row < hq ? (const T*)q.x + ahead.t * q.xt + row * q.xh : (const T*)k.x + ahead.t * k.xt + (row - hq) * k.xh;
                    sm100::cp_async_16(sm100::smem_u32(&ring[stage][u][0][lane]), x + e0, 16);
                    sm100::cp_async_16(sm100::smem_u32(&ring[stage][u][1][lane]), x + e1, 16);
                }
            }
            next(ahead);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < AHEAD - 1; ++i) fetch(i);
    int stage = 0;
    int64_t shown = -1;  // the token whose angles are held
    float2 sn[4], cs[4];
    while (at.item < items) {
        const int64_t t = at.t;
        if (t != shown) {
            shown = t;
            const double pos = (double)__ldg(position + t);
            double f = turn0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                sn[j] = sf::f2(0.f);
                cs[j] = sf::f2(1.f);
                if (turned) {
                    sincos_turns(pos * f, &sn[j].x, &cs[j].x);
                    f *= ratio;
                    sincos_turns(pos * f, &sn[j].y, &cs[j].y);
                    f *= ratio;
                }
            }
        }
        // Into the place that the last pair left, whose values have been used.
        fetch(stage == 0 ? AHEAD - 1 : stage - 1);
        asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD - 1) : "memory");
        uint4 a[2], b[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            a[u] = b[u] = make_uint4(0, 0, 0, 0);
            if (row_of(at, u) >= 0) {
                a[u] = ring[stage][u][0][lane];
                b[u] = ring[stage][u][1][lane];
            }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int row = row_of(at, u);
            float2 va[4], vb[4];
            unpack8<T>(a[u], va);
            unpack8<T>(b[u], vb);
            float2 ss = sf::f2_mul(va[0], va[0]);
#pragma unroll
            for (int j = 1; j < 4; ++j) ss = sf::f2_fma(va[j], va[j], ss);
#pragma unroll
            for (int j = 0; j < 4; ++j) ss = sf::f2_fma(vb[j], vb[j], ss);
            float sum = ss.x + ss.y;
#pragma unroll
            for (int o = LPR / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (row < 0) continue;
            const float2 rs = sf::f2(rsqrtf(fmaf(sum, inv_d, eps)));
            const bool isq = row < hq;
            float2 w0[4], w1[4], o0[4], o1[4];
            unpack8<T>(w_s[isq ? 0 : 1][0][p], w0);
            unpack8<T>(w_s[isq ? 0 : 1][1][p], w1);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 y0 = sf::f2_mul(sf::f2_mul(va[j], rs), w0[j]), y1 = sf::f2_mul(sf::f2_mul(vb[j], rs), w1[j]);
                o0[j] = y0;
                o1[j] = y1;
                if (turned) {  // where nothing turns an infinite partner would leave NaN
                    o0[j] = make_float2(fmaf(-y1.x, sn[j].x, y0.x * cs[j].x), fmaf(-y1.y, sn[j].y, y0.y * cs[j].y));
                    o1[j] = sf::f2_fma(y1, cs[j], sf::f2_mul(y0, sn[j]));
                }
            }
            T* y = isq ? (T*)q.y + t * q.yt + row * q.yh : (T*)k.y + t * k.yt + (row - hq) * k.yh;
            *reinterpret_cast<uint4*>(y + e0) = pack8<T>(o0);
            *reinterpret_cast<uint4*>(y + e1) = pack8<T>(o1);
        }
        stage = stage + 1 == AHEAD ? 0 : stage + 1;
        next(at);
    }
}

// Any D, rotary size and 2-byte alignment: a warp a row, element by element.  A lane reads and
// writes both members of its pairs, so in-place calls stay right here too.
template <typename T>
__global__ void __launch_bounds__(256) qk_norm_rope_general_kernel(const Side q, const Side k, const int32_t* __restrict__ position,
                                                                   int64_t tokens, int hq, int hk, int D, int r, double base, float eps) {
    const int lane = threadIdx.x & 31;
    const int64_t rows = tokens * (hq + hk);
    const int64_t step = (int64_t)gridDim.x * (blockDim.x >> 5);
    for (int64_t i = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); i < rows; i += step) {
        const int64_t t = i / (hq + hk);
        const int row = (int)(i - t * (hq + hk));
        const Side& s = row < hq ? q : k;
        const int64_t h = row < hq ? row : row - hq;
        const T* x = (const T*)s.x + t * s.xt + h * s.xh;
        T* y = (T*)s.y + t * s.yt + h * s.yh;
        const T* w = (const T*)s.w;
        float sum = 0.f;
        for (int d = lane; d < D; d += 32) {
            const float v = sf::Dt<T>::to_f(x[d]);
            sum = fmaf(v, v, sum);
        }
        const float rs = rsqrtf(sf::warp_sum(sum) / (float)D + eps);
        const double pos = (double)position[t];
        for (int d = lane; d < r; d += 32) {
            const float y0 = sf::Dt<T>::to_f(x[d]) * rs * sf::Dt<T>::to_f(w[d]);
            const float y1 = sf::Dt<T>::to_f(x[d + r]) * rs * sf::Dt<T>::to_f(w[d + r]);
            float sn, cs;
            sincos_turns(pos * (pow(base, -(double)d / (double)r) * 0.15915494309189533577), &sn, &cs);
            y[d] = sf::Dt<T>::from_f(y0 * cs - y1 * sn);
            y[d + r] = sf::Dt<T>::from_f(y0 * sn + y1 * cs);
        }
        for (int d = 2 * r + lane; d < D; d += 32) y[d] = sf::Dt<T>::from_f(sf::Dt<T>::to_f(x[d]) * rs * sf::Dt<T>::to_f(w[d]));
    }
}

template <typename T, int LPR>
int launch_vec(const Side& q, const Side& k, const int32_t* pos, int64_t T_, int hq, int hk, int D, int r, double base, float eps,
               cudaStream_t st, char* err, uint64_t cap) {
    constexpr int RPW = 32 / LPR;
    const int64_t ctas = (int64_t)sf::sm_count() * CTAS;
    const int64_t groups = (hq + hk + RPW - 1) / RPW;
    // A warp takes a whole token (its angles once) while the tokens fill the GPU's warps; fewer
    // tokens are split over their heads so that every warp has work.
    int64_t parts = ctas * WARPS / T_;
    parts = parts < 1 ? 1 : (parts > groups ? groups : parts);
    const int64_t items = T_ * parts;
    // Small problems: two-warp CTAs spread over all SMs.
    const int threads = items <= (int64_t)sf::sm_count() * 8 ? 64 : 32 * WARPS;
    int64_t blocks = (items + threads / 32 - 1) / (threads / 32);
    if (blocks > ctas * (32 * WARPS / threads)) blocks = ctas * (32 * WARPS / threads);
    qk_norm_rope_kernel<T, LPR><<<(unsigned)blocks, threads, 0, st>>>(q, k, pos, T_, hq, hk, D, r, r ? std::pow(base, -1.0 / (double)r) : 1.0, eps,
                                                                      (int)parts);
    return sf::check_launch("qk_norm_rope launch", err, cap);
}

bool vec_side(const Side& s, int64_t T_, int64_t h) {
    if (h == 0) return true;
    return sf::aligned16(s.x) && sf::aligned16(s.y) && sf::aligned16(s.w) && (T_ == 1 || (s.xt % 8 == 0 && s.yt % 8 == 0)) &&
           (h == 1 || (s.xh % 8 == 0 && s.yh % 8 == 0));
}

template <typename T>
int launch_t(const Side& q, const Side& k, const int32_t* pos, int64_t T_, int hq, int hk, int D, int rotary, double base, float eps,
             int32_t variant, cudaStream_t st, char* err, uint64_t cap) {
    const int r = rotary / 2;
    const bool vec = D % 16 == 0 && D <= 512 && r % 8 == 0 && vec_side(q, T_, hq) && vec_side(k, T_, hk);
    if (variant == 1 && !vec)
        return sf::fail(SF_EINVAL, err, cap, "qk_norm_rope: the vectorised variant needs D %% 16 == 0, D <= 512, rotary %% 16 == 0 and 16-byte aligned rows");
    if (vec && variant != 2) {
        if (D <= 64) return launch_vec<T, 4>(q, k, pos, T_, hq, hk, D, r, base, eps, st, err, cap);
        if (D <= 128) return launch_vec<T, 8>(q, k, pos, T_, hq, hk, D, r, base, eps, st, err, cap);
        if (D <= 256) return launch_vec<T, 16>(q, k, pos, T_, hq, hk, D, r, base, eps, st, err, cap);
        return launch_vec<T, 32>(q, k, pos, T_, hq, hk, D, r, base, eps, st, err, cap);
    }
    const int64_t rows = T_ * (hq + hk);
    int64_t blocks = (rows + 7) / 8;
    const int64_t most = (int64_t)sf::sm_count() * 8;
    if (blocks > most) blocks = most;
    qk_norm_rope_general_kernel<T><<<(unsigned)blocks, 256, 0, st>>>(q, k, pos, T_, hq, hk, D, r, base, eps);
    return sf::check_launch("qk_norm_rope general launch", err, cap);
}

}  // namespace

extern "C" int sf_qk_norm_rope(const sf_qk_norm_rope_args* x, void* stream, char* err, uint64_t cap) {
    if (!x) return sf::fail(SF_EINVAL, err, cap, "qk_norm_rope: null arguments");
    const int64_t T = x->T, Hq = x->Hq, Hk = x->Hk, D = x->D;
    if (T < 0 || Hq < 0 || Hk < 0 || Hq + Hk > (1 << 20) || D < 1 || D > (1 << 20))
        return sf::fail(SF_EINVAL, err, cap, "qk_norm_rope: need T, Hq, Hk >= 0 and D >= 1");
    if (x->variant < 0 || x->variant > 2) return sf::fail(SF_EINVAL, err, cap, "qk_norm_rope: no variant %d", x->variant);
    if (x->rotary < 0 || x->rotary % 2 || x->rotary > D) return sf::fail(SF_EINVAL, err, cap, "qk_norm_rope: rotary must be even and at most D");
    if (!(x->base > 0) || !std::isfinite(x->base)) return sf::fail(SF_EINVAL, err, cap, "qk_norm_rope: base must be > 0");
    if (!(x->eps >= 0)) return sf::fail(SF_EINVAL, err, cap, "qk_norm_rope: eps must be >= 0");
    if (x->dtype != SF_DTYPE_F16 && x->dtype != SF_DTYPE_BF16)
        return sf::fail(SF_EINVAL, err, cap, "qk_norm_rope: dtype %d is not fp16/bf16", x->dtype);
    for (const sf_rows* r : {&x->q_rows, &x->k_rows, &x->q_out_rows, &x->k_out_rows})
        if (r->token < 0 || r->head < 0) return sf::fail(SF_EINVAL, err, cap, "qk_norm_rope: negative stride");
    if (T * (Hq + Hk) == 0) return SF_OK;
    if (!x->positions || (Hq && (!x->q || !x->q_out || !x->wq)) || (Hk && (!x->k || !x->k_out || !x->wk)))
        return sf::fail(SF_EINVAL, err, cap, "qk_norm_rope: null tensor pointer");
    const Side q{x->q, x->q_out, x->wq, x->q_rows.token, x->q_rows.head, x->q_out_rows.token, x->q_out_rows.head};
    const Side k{x->k, x->k_out, x->wk, x->k_rows.token, x->k_rows.head, x->k_out_rows.token, x->k_out_rows.head};
    const int32_t* pos = (const int32_t*)x->positions;
    if (x->dtype == SF_DTYPE_F16)
        return launch_t<__half>(q, k, pos, T, (int)Hq, (int)Hk, (int)D, (int)x->rotary, x->base, (float)x->eps, x->variant, (cudaStream_t)stream, err, cap);
    return launch_t<__nv_bfloat16>(q, k, pos, T, (int)Hq, (int)Hk, (int)D, (int)x->rotary, x->base, (float)x->eps, x->variant, (cudaStream_t)stream, err,
                                   cap);
}
