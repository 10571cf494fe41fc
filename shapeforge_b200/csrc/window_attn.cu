// Attention of packed prompts with grouped heads, a sliding window and sinks, sm_100a:
//
//   o[i, h, :] = sum_j softmax_j(scale q[i, h, :] . k[j, h / g, :]) v[j, h / g, :]
//   query i of a sequence with nq queries and nk keys sits at position p = i + nk - nq and sees the
//   keys j <= p with j > p - window or j < sinks (window 0: all j <= p)
//
// q, o [Tq, Hq, D] and k, v [Tk, Hk, D] with any token and head strides, g = Hq / Hk, sequences packed
// by cu_seqlens; fp16 / bf16, softmax statistics in fp32, weights in some 16 (bf16) or 22 (fp16) bits.  A query that sees nothing gives zeros; rows
// of no sequence are left as they were.
#include "sf_common.cuh"
#include "sm100.cuh"
#include "tma_host.cuh"

#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <mutex>
#include <type_traits>

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
    int slots;           // of tokens, a kv head
    int splits;          // CTAs that share the keys of a pair of row tiles; above 1 each leaves its state for the join:
    int whole;           // pairs of row tiles, in the grid's order, whose keys stay together all the same
    // [splits][rows][D] unnormalised outputs, [splits][rows][2] running max, sum; the rows are the tensor's [tq][heads],
    // or with whole > 0 only those of the other pairs, in the grid's order.
    float *part, *stat;
};

// Keys [0, sinks) and [low, high) of a query at position p.
struct Keys {
    int sinks, low, high;
    __device__ __forceinline__ Keys(const Args& a, int p) {
        high = max(0, p + 1);
        low = a.window ? max(0, max(0, p) - a.window + 1) : 0;  // a position far below 0 less a large window wraps
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

// ---- tensor-core kernel: D 64 / 128 ----------------------------------------------------------------
//
// The query heads of a kv head share its keys, so a tile's 128 rows are (token, head of the group) pairs:
// TQ = 128 / g tokens with their g heads.  A window then costs a tile g times less padding, and short
// prompts fill their rows.  A CTA takes two such tiles of consecutive tokens over one stream of key tiles
// (each key and value tile is fetched once for 256 rows) and owns an SM:
//   warp 0        TMA producer: both Q tiles, then K_j and V_j tiles of up to 128 keys, two slots each;
//   warp 1        MMA issuer, in the order P0.V(j-1), S0(j), P1.V(j-1), S1(j): one tile's products run
//                 under the other's softmax; S (then P over it) and O of both tiles fill TMEM.  (An
//                 issuer a tile let both tiles wait, then compute, at the same time: 498 against 402 us
//                 at 16384 tokens, window 4096, 16 heads on 2, without P's residual.)  Its operands are kept uniform over the
//                 warp: issued from one divergent lane a product cost ~130 cycles against the pipe's 64;
//   warp 2        zeroes the value rows behind a sequence's last key (0 times another sequence's NaN or
//                 infinity would be NaN) and hands the tile on;
//   warps 4..7    softmax of tile 0, a thread a row; warps 8..11 of tile 1.
// Key tiles begin at the first key that the CTA's first token sees (a TMA coordinate along the tokens
// needs no alignment), and the sinks in front of it are a tile of their own; a tile of n keys costs
// n rounded up to 16 in both products and 32 in the softmax.  Tiles that every row sees in full skip the
// mask.  Running max and sum in fp32; the max follows a score only past 2^8, so O is rarely rescaled.
// P goes into its product twice, as a 16-bit high part and the 16-bit residual, over the columns that its scores
// leave, as in this library's other attention: rounded once to bf16, it moved results by half a step of the type
// (and took 381 us where the two take 522).
// 16384 tokens, 16 heads on 2 of 128, window 4096, bf16: 522 us, 922 TFLOP/s of seen scores (56 % of what a large
// library product reaches; 84 % with P . V counted twice): a step of 128 keys for 256 rows takes 1.9 us, its products
// 1.56 at the pipe's rate.  P's first hand-over at 32, 64 or 96 keys: 527, 523, 522.  1203 tokens in 9 prompts, window
// 128: 22 us, two CTAs in turn on an SM, latency.  (Without the residual, CTAs that take their next piece from the
// hardware's scheduler hid the start and end, but the registers that cost the softmax slowed every step: 411 us.)
// A row that comes out NaN or infinite may have that from values that it does not see, which share its tiles and which
// a weight of zero does not silence.  If its softmax sum is not finite the scores it sees are not, and all of it is NaN;
// else `settle` looks through the values that the warp's rows see, once for all of them: a column that sees a NaN or an
// infinity is that, and a row with some other column of that kind is computed again key by key.  So only rows within a
// tile or two of a bad value that they do not see are (16384 causal tokens of 16 heads on 2: 1.1 ms, 5.6 with
// the first value infinite, 1.1 with the first key NaN).

constexpr int BOX = 128 * 128;       // 128 rows of 64 16-bit elements
constexpr int TC_THREADS = 384;
constexpr int FIRST_KEYS = 96;       // keys of a tile whose P is handed over first, then the rest
constexpr uint32_t O_COL = 256;      // S / P of tile t at column 128 t, O at 256 + 128 t

__device__ sm100::KernelStatus g_window_status;

struct __align__(8) Bars {
    uint64_t q_full[2];
    uint64_t k_full[2], k_empty[2];
    uint64_t v_full[2], v_ready[2], v_empty[2];
    uint64_t s_full[2], p_full[2][2], o_done[2];
    uint32_t tmem_base;
};

template <int D>
struct Layout {
    static constexpr int DB = D / 64;
    static constexpr int TILE = DB * BOX;
    static constexpr int Q = 0;              // [2]
    static constexpr int K = 2 * TILE;       // [2]
    static constexpr int V = 4 * TILE;       // [2]
    static constexpr int BARS = 6 * TILE;
    static constexpr int BYTES = BARS + 256;
};

// A value that all lanes share, told to the compiler: what is computed from it, loops and branches
// included, can run on the uniform datapath, where the tensor instructions take their operands from.
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }

// The key tiles of a CTA: sinks [0, sink_end), then [low, high) in steps of 128; of these the n from `base` on
// are this split's (tile j below is j - base of the CTA's own).
struct Walk {
    int sink_end, sink_tiles, low, high, base, n;
    __device__ __forceinline__ bool in_sinks(int j) const { return j + base < sink_tiles; }
    __device__ __forceinline__ int start(int j) const { return in_sinks(j) ? 128 * (j + base) : low + 128 * (j + base - sink_tiles); }
};

// What one of the CTA's two row tiles makes of them.
struct Span {
    int first, last;  // positions of its first and last token (last < 0: no token that sees a key)
    int skip;         // the window's first tile is left out (it ends before the tile's own window)
    int end;          // keys below this are seen by some row
    int front;        // keys from here on are inside every row's window
    __device__ __forceinline__ Span(const Args& a, const Walk& w, int first_, int tokens) {
        first = first_;
        last = tokens > 0 ? first_ + tokens - 1 : -1;
        end = min(w.high, last + 1);
        front = a.window ? last - a.window + 1 : 0;
        skip = a.window && last >= 0 && w.low + 128 <= max(0, first) - a.window + 1 && w.low >= a.sinks ? 1 : 0;
    }
    // Keys [0, count) of tile j can be seen.
    __device__ __forceinline__ int count(const Walk& w, int j) const { return max(0, min(128, (w.in_sinks(j) ? w.sink_end : end) - w.start(j))); }
    __device__ __forceinline__ bool active(const Walk& w, int j) const {
        return last >= 0 && (w.in_sinks(j) || (w.start(j) < end && !(skip && j + w.base == w.sink_tiles)));
    }
    // Every row sees all 128 keys of tile j.
    __device__ __forceinline__ bool full(const Walk& w, int j, int sinks) const {
        const int s = w.start(j);
        return w.in_sinks(j) ? s + 128 <= w.sink_end : s + 127 <= first && (s >= front || s + 128 <= sinks);
    }
};

// Where a CTA's tokens lie: its sequence's rows and keys, its first token and that one's position.
struct Where {
    int qe, kb, ke, tok0, pos0;
};
// Sequence i owns the slots from cu_q[i] / TT + i on, TT tokens each, which leaves out no token whatever the
// lengths and needs no prefix of tile counts; false: a slot without tokens.  Every lane of the warp.
__device__ __forceinline__ bool locate(const Args& a, int TT, int slot, Where* w) {
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = a.seqs, qb = 0;
    while (true) {
        const int step = max(1, (hi - lo + 31) >> 5);
        const int i = min(lo + lane * step, a.seqs);
        const int q_here = __ldg(a.cu_q + i), k_here = step == 1 ? __ldg(a.cu_k + i) : 0;
        const bool here = lo + lane * step < hi && min(max(0, q_here), (int)a.tq) / TT + i <= slot;
        const uint32_t yes = __ballot_sync(0xffffffffu, here);
        const int k = yes ? 31 - __clz(yes) : 0;
        if (step > 1) {
            lo = lo + k * step;
            hi = min(hi, lo + step);
            continue;
        }
        // The bounds come from the lanes k and k + 1.
        const int top_q = k < 31 ? __shfl_sync(0xffffffffu, q_here, min(k + 1, 31)) : __ldg(a.cu_q + lo + 32);
        const int top_k = k < 31 ? __shfl_sync(0xffffffffu, k_here, min(k + 1, 31)) : __ldg(a.cu_k + lo + 32);
        qb = min(max(0, __shfl_sync(0xffffffffu, q_here, k)), (int)a.tq);
        w->qe = max(qb, min(top_q, (int)a.tq));
        w->kb = min(max(0, __shfl_sync(0xffffffffu, k_here, k)), (int)a.tk);
        w->ke = max(w->kb, min(top_k, (int)a.tk));
        lo += k;
        break;
    }
    const int64_t at = qb + (int64_t)(slot - qb / TT - lo) * TT;
    if (at < qb || at >= w->qe) return false;
    w->tok0 = uniform((int)at);
    w->pos0 = (w->tok0 - qb) + (w->ke - w->kb) - (w->qe - qb);
    return true;
}

// Bits [0, n) of a 32-bit word.
__device__ __forceinline__ uint32_t below(int n) { return n <= 0 ? 0u : (n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1u); }

__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// The products' tcgen05.mma, issued by the one lane with `lead`, as predicated instructions of a warp that
// runs together: descriptors and addresses then stay in uniform registers, and several go into one block
// that forms the predicate once.  A descriptor is given as its two words; offsets go onto the address
// field of the lower one.
#define SF_DESC(reg, lo, hi, off) "add.u32 x, " lo ", " off ";\nmov.b64 " reg ", {x, " hi "};\n"
#define SF_QK_STEP(off, acc) SF_DESC("da", "%1", "%2", off) SF_DESC("db", "%3", "%4", off) "@q tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, " acc ";\n"
#define SF_QK_BEGIN "{\n.reg .pred p, f, q;\n.reg .b32 x;\n.reg .b64 da, db;\nsetp.ne.b32 q, %6, 0;\nsetp.eq.b32 p, %6, %6;\nsetp.ne.b32 f, %6, %6;\n"
#define SF_QK_ARGS(d, a, b, idesc, lead) \
    "r"(d), "r"((uint32_t)(a)), "r"((uint32_t)((a) >> 32)), "r"((uint32_t)(b)), "r"((uint32_t)((b) >> 32)), "r"(idesc), "r"(lead)
// S = Q . K^T, D / 16 products; in a tile of 128 rows 16 elements of D are 2 on in the address field, 64 are a box.
template <int D>
__device__ __forceinline__ void issue_qk(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t lead) {
    if constexpr (D == 128) {
        asm volatile(SF_QK_BEGIN SF_QK_STEP("0", "f") SF_QK_STEP("2", "p") SF_QK_STEP("4", "p") SF_QK_STEP("6", "p") SF_QK_STEP("1024", "p")
                         SF_QK_STEP("1026", "p") SF_QK_STEP("1028", "p") SF_QK_STEP("1030", "p") "}\n" ::SF_QK_ARGS(d, a, b, idesc, lead)
                     : "memory");
    } else {
        asm volatile(SF_QK_BEGIN SF_QK_STEP("0", "f") SF_QK_STEP("2", "p") SF_QK_STEP("4", "p") SF_QK_STEP("6", "p") "}\n" ::SF_QK_ARGS(d, a, b, idesc, lead)
                     : "memory");
    }
}
// O += P . V over 32 keys or over 16.  P of 32 keys lies in 32 columns: the high parts in the first 16, the
// residuals behind them; 16 keys of V are 128 on.
#define SF_PV_STEP(col, off, acc) "add.u32 y, %1, " col ";\n" SF_DESC("db", "%2", "%3", off) "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [y], db, %4, " acc ";\n"
__device__ __forceinline__ void issue_pv32(uint32_t d, uint32_t p, uint64_t v, uint32_t idesc, uint32_t accumulate, uint32_t lead) {
    asm volatile("{\n.reg .pred p, f, q;\n.reg .b32 x, y;\n.reg .b64 db;\nsetp.ne.b32 q, %6, 0;\nsetp.eq.b32 p, %6, %6;\nsetp.ne.b32 f, %5, 0;\n" SF_PV_STEP(
                     "0", "0", "f") SF_PV_STEP("8", "128", "p") SF_PV_STEP("16", "0", "p") SF_PV_STEP("24", "128", "p") "}\n" ::"r"(d),
                 "r"(p), "r"((uint32_t)v), "r"((uint32_t)(v >> 32)), "r"(idesc), "r"(accumulate), "r"(lead)
                 : "memory");
}
__device__ __forceinline__ void issue_pv16(uint32_t d, uint32_t p, uint64_t v, uint32_t idesc, uint32_t accumulate, uint32_t lead) {
    asm volatile("{\n.reg .pred p, f, q;\n.reg .b32 x, y;\n.reg .b64 db;\nsetp.ne.b32 q, %6, 0;\nsetp.eq.b32 p, %6, %6;\nsetp.ne.b32 f, %5, 0;\n" SF_PV_STEP(
                     "0", "0", "f") SF_PV_STEP("16", "0", "p") "}\n" ::"r"(d),
                 "r"(p), "r"((uint32_t)v), "r"((uint32_t)(v >> 32)), "r"(idesc), "r"(accumulate), "r"(lead)
                 : "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar, uint32_t lead) {
    asm volatile(
        "{\n"
        ".reg .pred q;\n"
        "setp.ne.b32 q, %1, 0;\n"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n"
        "}\n" ::"r"(sm100::smem_u32(bar)),
        "r"(lead)
        : "memory");
}

// mbar_wait for the hand-overs between products and softmax: reading the clock for the time limit costs some
// hundred cycles, so it begins only after waits that together outlast any product.
__device__ __forceinline__ bool wait_soon(uint64_t* bar, uint32_t parity, sm100::KernelStatus* st, uint32_t where) {
#pragma unroll 1
    for (int i = 0; i < 256; ++i)
        if (sm100::mbar_try_wait(bar, parity)) return true;
    return sm100::mbar_wait(bar, parity, st, where);
}

// Running state of a row: `m` the max that weights are relative to (log2 units), `l` their sum.
// An fp16 weight is held times 2^7: at most 2^15, and 2^-32 of the running max is still a half step of its
// smallest residual; `l` and O carry the same factor, which the division takes out.
template <typename T>
constexpr float LIFT = std::is_same<T, __half>::value ? 7.f : 0.f;
struct RowState {
    float m, l;
    // Take in a tile's row max; O (in TMEM) is rescaled when the max has grown by more than 2^8.
    template <typename T, int D>
    __device__ __forceinline__ float raise(float rmax, float scale_log2, uint32_t tmem_o, bool some) {
        const float m_new = max3_nan(m, rmax * scale_log2, m);
        const bool need = !(m_new <= m + 8.0f);
        if (some) {
            if (__any_sync(0xffffffffu, need)) {
                const float alpha = need ? exp2f(m - m_new) : 1.0f;
#pragma unroll 1
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t r[32];
                    sm100::tmem_ld_32x32b_x32(tmem_o + (uint32_t)(32 * c), r);
                    sm100::tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * alpha);
                    sm100::tmem_st_32x32b_x32(tmem_o + (uint32_t)(32 * c), r);
                }
                l *= alpha;
            }
        }
        if (need) m = m_new;
        return m == -INFINITY ? 0.f : m - LIFT<T>;
    }
};

// 32 scores to weights, adding them up: 16 words of high parts, then 16 of what they leave out, so that P . V is a
// product with P to some 16 (bf16) or 22 (fp16) bits.  A bf16 high part is the upper half of the fp32 word
// (one byte permute for two weights); the residual is exact before its own rounding.
template <typename T>
__device__ __forceinline__ void weights32(const uint32_t* r, float scale_log2, float m, float2 (&acc)[2], uint32_t (&w)[32]) {
    const float2 sc = sf::f2(scale_log2), nm = sf::f2(-m), minus = sf::f2(-1.f);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float2 x = sf::f2_fma(make_float2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])), sc, nm);
        const float2 p = make_float2(sf::ex2_ftz(x.x), sf::ex2_ftz(x.y));
        acc[i & 1] = sf::f2_add(acc[i & 1], p);
        float2 high;
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {
            const uint32_t a = __float_as_uint(p.x), b = __float_as_uint(p.y);
            w[i] = __byte_perm(a, b, 0x7632);
            high = make_float2(__uint_as_float(a & 0xFFFF0000u), __uint_as_float(b & 0xFFFF0000u));
        } else {
            w[i] = sf::Pair<T>::from_f2(p);
            high = sf::Pair<T>::to_f2(w[i]);
        }
        w[16 + i] = sf::Pair<T>::from_f2(sf::f2_fma(high, minus, p));
    }
}

__device__ __forceinline__ float max32(const uint32_t* r, float m) {
    float a[2] = {m, -INFINITY};
#pragma unroll
    for (int i = 0; i < 32; i += 4) {
        a[0] = max3_nan(a[0], __uint_as_float(r[i]), __uint_as_float(r[i + 1]));
        a[1] = max3_nan(a[1], __uint_as_float(r[i + 2]), __uint_as_float(r[i + 3]));
    }
    return max3_nan(a[0], a[1], a[1]);
}

// The rows of a warp whose output (written, at `out`) is not finite although their softmax sum is: lanes with `again`,
// each with its row's position and query row.  Values in 16-byte aligned rows, as the kernel below takes them.
template <typename T, int D>
__device__ __forceinline__ void settle(const Args& a, bool again, int p, int64_t kbegin, int64_t qrow, int head, T* out) {
    constexpr int E = D / 32, W = E / 2;  // the lane's columns E lane .. E lane + E - 1, two a word
    constexpr uint32_t EXP = std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
    const int lane = threadIdx.x & 31;
    uint32_t todo = __ballot_sync(0xffffffffu, again);
    if (!todo) return;
    const int kvh = __shfl_sync(0xffffffffu, head, __ffs(todo) - 1) / a.group;
    const T* v = (const T*)a.v + kbegin * a.vt + (int64_t)kvh * a.vh + E * lane;
    const Keys mine(a, again ? p : -1);
    const Keys all(a, -__reduce_max_sync(0xffffffffu, again ? -p : -0x7fffffff));  // of the first of them, but up to
    const int high = __reduce_max_sync(0xffffffffu, mine.high);                    // what the last sees
    const int n = all.sinks + high - all.low;
    // What the lane's row sees in column E l + e: bit l of [e].
    uint32_t nan[E] = {}, pos[E] = {}, neg[E] = {};
    constexpr int AHEAD = 8;
#pragma unroll 1
    for (int i0 = 0; i0 < n; i0 += AHEAD) {
        uint32_t x[AHEAD][W];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int i = min(i0 + u, n - 1);
            const T* row = v + (int64_t)(i < all.sinks ? i : all.low + (i - all.sinks)) * a.vt;
            if constexpr (W == 2) *reinterpret_cast<uint2*>(x[u]) = *reinterpret_cast<const uint2*>(row);
            else x[u][0] = *reinterpret_cast<const uint32_t*>(row);
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            bool bad = false;
#pragma unroll
            for (int k = 0; k < W; ++k) bad |= (x[u][k] & EXP) == EXP || (x[u][k] >> 16 & EXP) == EXP;
            if (!__any_sync(0xffffffffu, bad)) continue;
            const int i = min(i0 + u, n - 1), j = i < all.sinks ? i : all.low + (i - all.sinks);
            const bool sees = j < mine.sinks || (j >= mine.low && j < mine.high);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const uint32_t y = x[u][e / 2] >> (16 * (e & 1)) & 0xFFFFu;
                const bool special = (y & EXP) == EXP, is_nan = (y & 0x7FFFu) > EXP;
                const uint32_t b_nan = __ballot_sync(0xffffffffu, is_nan), b_pos = __ballot_sync(0xffffffffu, special && !is_nan && !(y >> 15)),
                               b_neg = __ballot_sync(0xffffffffu, special && !is_nan && y >> 15);
                if (sees) nan[e] |= b_nan, pos[e] |= b_pos, neg[e] |= b_neg;
            }
        }
    }
    for (; todo; todo &= todo - 1) {
        const int src = __ffs(todo) - 1;
        T* o = reinterpret_cast<T*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(out), src)) + E * lane;
        bool left = false;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const uint32_t here = __shfl_sync(0xffffffffu, nan[e], src) >> lane & 1u, up = __shfl_sync(0xffffffffu, pos[e], src) >> lane & 1u,
                           down = __shfl_sync(0xffffffffu, neg[e], src) >> lane & 1u;
            if (here | up | down) o[e] = sf::Dt<T>::from_f(here || (up && down) ? NAN : (up ? INFINITY : -INFINITY));
            else left |= !(fabsf(sf::Dt<T>::to_f(o[e])) < INFINITY);
        }
        if (__any_sync(0xffffffffu, left)) {
            __syncwarp();
            row_by_warp<T>(a, D, __shfl_sync(0xffffffffu, (long long)qrow, src), __shfl_sync(0xffffffffu, head, src), kbegin,
                           __shfl_sync(0xffffffffu, p, src), o - E * lane);
        }
    }
}

// LINE: a.whole pairs of row tiles keep their keys, the others are split, all in one line of CTAs.
template <typename T, int D, bool LINE>
__global__ void __launch_bounds__(TC_THREADS, 1)
    window_tc_kernel(const __grid_constant__ Args a, const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mk16,
                     const __grid_constant__ CUtensorMap mv, const __grid_constant__ CUtensorMap mv16, int tq_tile) {
    using L = Layout<D>;
    constexpr int DB = L::DB;
    constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    Bars* bars = reinterpret_cast<Bars*>(smem + L::BARS);
    sm100::KernelStatus* status = &g_window_status;
    const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    // The whole pairs, then the others' first parts, their second parts and so on.
    const int rest = LINE ? a.slots * (a.heads / a.group) - a.whole : 1;
    const int part = !LINE ? blockIdx.z : (blockIdx.x < a.whole ? 0 : (blockIdx.x - a.whole) / rest);
    const int parts = LINE && blockIdx.x < a.whole ? 1 : a.splits;
    const int pair = LINE ? blockIdx.x - part * rest : 0;
    const int kvh = LINE ? pair / a.slots : blockIdx.y;

    // Set-up that needs no lengths runs while the search below waits for them.
    if (threadIdx.x == 0) {
        for (const CUtensorMap* m : {&mq, &mk, &mk16, &mv, &mv16}) sm100::tma_prefetch_desc(m);
        for (int i = 0; i < 2; ++i) {
            sm100::mbar_init(&bars->q_full[i], 1);
            sm100::mbar_init(&bars->k_full[i], 1);
            sm100::mbar_init(&bars->k_empty[i], 1);
            sm100::mbar_init(&bars->v_full[i], 1);
            sm100::mbar_init(&bars->v_ready[i], 32);
            sm100::mbar_init(&bars->v_empty[i], 1);
            sm100::mbar_init(&bars->s_full[i], 1);
            sm100::mbar_init(&bars->p_full[i][0], 128);
            sm100::mbar_init(&bars->p_full[i][1], 128);
            sm100::mbar_init(&bars->o_done[i], 1);
        }
        sm100::fence_mbar_init();
    }
    // Rows of the Q tiles that no copy writes.
    const int qrows = tq_tile * a.group;
    for (int i = threadIdx.x; i < 2 * DB * (128 - qrows) * 8; i += TC_THREADS) {
        const int box = i / ((128 - qrows) * 8), rest = i % ((128 - qrows) * 8);
        *reinterpret_cast<uint4*>(smem + L::Q + box * BOX + (qrows + rest / 8) * 128 + (rest % 8) * 16) = make_uint4(0, 0, 0, 0);
    }
    sm100::fence_proxy_async_smem();

    Where at;
    const bool found = locate(a, 2 * tq_tile, LINE ? a.slots - 1 - (pair - kvh * a.slots) : gridDim.x - 1 - blockIdx.x, &at);
    if (!found) return;  // a slot that rounding left over
    const int tok0 = at.tok0, kb = at.kb, ke = at.ke;
    const int rows_tok[2] = {min(tq_tile, at.qe - tok0), max(0, min(tq_tile, at.qe - tok0 - tq_tile))};
    const int pos0 = uniform(at.pos0);
    Walk w;
    w.high = max(0, pos0 + uniform(rows_tok[0] + rows_tok[1]));
    w.low = uniform(a.window ? max(0, max(0, pos0) - a.window + 1) : 0);
    w.sink_end = min(a.sinks, w.low);
    w.sink_tiles = (w.sink_end + 127) >> 7;
    w.n = w.high > 0 ? w.sink_tiles + ((w.high - w.low + 127) >> 7) : 0;
    w.base = 0;
    if (parts > 1) {
        const int n = w.n;
        w.base = (int)((int64_t)n * part / parts);
        w.n = (int)((int64_t)n * (part + 1) / parts) - w.base;
    }
    const Span span0(a, w, pos0, uniform(rows_tok[0])), span1(a, w, pos0 + tq_tile, uniform(rows_tok[1]));

    if (warp == 1) {
        sm100::tmem_alloc(&bars->tmem_base, 512);
        sm100::tmem_relinquish();
    }
    sm100::tc_fence_before();
    __syncthreads();
    sm100::tc_fence_after();
    const uint32_t tmem = uniform(bars->tmem_base);

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
        if (warp == 0) {
            if (lane == 0 && w.n > 0) {
                for (int t = 0; t < 2; ++t) {
                    if ((t ? span1.last : span0.last) < 0) continue;
                    sm100::mbar_arrive_expect_tx(&bars->q_full[t], DB * qrows * 128);
                    for (int b = 0; b < DB; ++b)
                        sm100::tma_load_3d(smem + L::Q + (t * DB + b) * BOX, &mq, &bars->q_full[t], 64 * b, kvh * a.group, tok0 + t * tq_tile);
                }
                int keys_in = 0, values_in = 0;  // tiles whose copies were issued
                for (int j = 0; j < w.n; ++j) {
                    const int st = j & 1;
                    const uint32_t ph = (uint32_t)(j >> 1) & 1u;
                    // Keys that some tile multiplies, in whole 16s.
                    const int rows = (max(span0.count(w, j), span1.count(w, j)) + 15) & ~15;
                    const int key = kb + w.start(j);
                    for (int kv = 0; kv < 2; ++kv) {
                        uint64_t* empty = kv ? &bars->v_empty[st] : &bars->k_empty[st];
                        uint64_t* full = kv ? &bars->v_full[st] : &bars->k_full[st];
                        uint8_t* dst = smem + (kv ? L::V : L::K) + st * L::TILE;
                        if (!sm100::mbar_wait(empty, ph ^ 1u, status, 120 + kv)) goto fetched;
                        sm100::mbar_arrive_expect_tx(full, DB * rows * 128);
                        ++(kv ? values_in : keys_in);
                        for (int b = 0; b < DB; ++b) {
                            if (rows == 128) {
                                sm100::tma_load_3d(dst + b * BOX, kv ? &mv : &mk, full, 64 * b, kvh, key);
                            } else {
                                for (int r = 0; r < rows; r += 16)
                                    sm100::tma_load_3d(dst + b * BOX + r * 128, kv ? &mv16 : &mk16, full, 64 * b, kvh, key + r);
                            }
                        }
                    }
                }
            fetched:
                // No copy is in flight when the CTA ends, also after a wait that gave up.
                for (int t = 0; t < 2; ++t)
                    if ((t ? span1.last : span0.last) >= 0) sm100::mbar_wait(&bars->q_full[t], 0, nullptr, 0);
                for (int j = max(0, keys_in - 2); j < keys_in; ++j) sm100::mbar_wait(&bars->k_full[j & 1], (uint32_t)(j >> 1) & 1u, nullptr, 0);
                for (int j = max(0, values_in - 2); j < values_in; ++j) sm100::mbar_wait(&bars->v_full[j & 1], (uint32_t)(j >> 1) & 1u, nullptr, 0);
            }
        } else if (warp == 1) {
            if (w.n > 0) {
                const uint32_t lead = sm100::elect_one();
                constexpr uint32_t idesc_s = sm100::idesc_f16(128, 0, BF16);
                constexpr uint32_t idesc_o = sm100::idesc_f16_bmn(128, D, BF16);
                constexpr uint32_t NEXT = L::TILE >> 4;  // from one tile to the next in a descriptor's address field
                const uint64_t dq = sm100::smem_desc_k_sw128(sm100::smem_u32(smem + L::Q)), dk = sm100::smem_desc_k_sw128(sm100::smem_u32(smem + L::K)),
                               dv = sm100::smem_desc_mn_sw128(sm100::smem_u32(smem + L::V), BOX, 1024);
                // The lanes wait each for itself and agree once a step on whether a wait gave up.
                bool ok = true;
                auto wait = [&](uint64_t* bar, uint32_t parity, uint32_t where) { ok &= wait_soon(bar, parity, status, where); };
                // O_t += P_t(j) . V(j) over `keys` keys, the first of them as soon as their P is there.
                auto pv = [&](int t, int j, int keys, uint32_t turn) {
                    const uint64_t d = dv + (j & 1) * NEXT;
                    const uint32_t to = tmem + O_COL + 128u * t, tp = tmem + 128u * t;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        wait(&bars->p_full[t][h], turn & 1u, 123);
                        __syncwarp();
                        sm100::tc_fence_after();
#pragma unroll
                        for (int c = h ? FIRST_KEYS / 32 : 0; c < (h ? 4 : FIRST_KEYS / 32); ++c) {
                            if (keys > 32 * c + 16) issue_pv32(to, tp + 32u * c, d + 256 * c, idesc_o, c > 0 || turn > 0 ? 1u : 0u, lead);
                            else if (keys > 32 * c) issue_pv16(to, tp + 32u * c, d + 256 * c, idesc_o, c > 0 || turn > 0 ? 1u : 0u, lead);
                        }
                    }
                };
                // S_t(j) = Q_t . K(j)^T over the columns that P_t was read from (the pipe runs this thread's
                // products in order).
                auto qk = [&](int t, int j, int keys) {
                    issue_qk<D>(tmem + 128u * t, dq + t * NEXT, dk + (j & 1) * NEXT, idesc_s | ((uint32_t)((keys + 15) >> 4) << 18), lead);
                    commit(&bars->s_full[t], lead);
                };
                // A step between two tiles of 128 keys for both row tiles, key tile j in slot ST: nothing to
                // decide, since every instruction here is on the way from one softmax to the next.
                uint32_t turns0 = 0, turns1 = 0;  // tiles of P consumed
                auto whole_step = [&](auto slot, uint32_t k_parity, uint32_t v_parity) {
                    constexpr int ST = decltype(slot)::value;
                    const uint64_t v = dv + (1 - ST) * NEXT, k = dk + ST * NEXT;
                    constexpr uint32_t idesc = sm100::idesc_f16(128, 128, BF16);
                    wait(&bars->v_ready[1 - ST], v_parity, 122);
                    wait(&bars->k_full[ST], k_parity, 125);
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        const uint32_t turn = t ? turns1 : turns0, to = tmem + O_COL + 128u * t, tp = tmem + 128u * t;
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            wait(&bars->p_full[t][h], turn & 1u, 123);
                            __syncwarp();
                            sm100::tc_fence_after();
#pragma unroll
                            for (int c = h ? FIRST_KEYS / 32 : 0; c < (h ? 4 : FIRST_KEYS / 32); ++c)
                                issue_pv32(to, tp + 32u * c, v + 256 * c, idesc_o, c > 0 || turn > 0 ? 1u : 0u, lead);
                        }
                        if (t == 1) commit(&bars->v_empty[1 - ST], lead);
                        issue_qk<D>(tp, dq + t * NEXT, k, idesc, lead);
                        commit(&bars->s_full[t], lead);
                    }
                    commit(&bars->k_empty[ST], lead);
                    ++turns0;
                    ++turns1;
                };
                // Tiles [whole0, whole1) have 128 keys for both.
                const int whole0 = w.sink_tiles + (span0.skip | span1.skip) - w.base;
                const int whole1 = span0.last >= 0 && span1.last >= 0 ? min(w.n, w.sink_tiles + (min(span0.end, span1.end) - w.low) / 128 - w.base) : 0;
                if (span0.last >= 0) wait(&bars->q_full[0], 0, 124);
                if (span1.last >= 0) wait(&bars->q_full[1], 0, 124);
                int keys0 = 0, keys1 = 0;         // of tile j - 1, 0: it is not for that row tile
                int j = 0;
                for (; j <= w.n; ++j) {
                    const int next0 = j < w.n && span0.active(w, j) ? span0.count(w, j) : 0, next1 = j < w.n && span1.active(w, j) ? span1.count(w, j) : 0;
                    if (j > 0) wait(&bars->v_ready[(j - 1) & 1], (uint32_t)((j - 1) >> 1) & 1u, 122);
                    if (keys0) pv(0, j - 1, keys0, turns0++);
                    if (j == w.n) commit(&bars->o_done[0], lead);
                    if (j < w.n) wait(&bars->k_full[j & 1], (uint32_t)(j >> 1) & 1u, 125);
                    __syncwarp();
                    sm100::tc_fence_after();
                    if (next0) qk(0, j, next0);
                    if (keys1) pv(1, j - 1, keys1, turns1++);
                    if (j == w.n) commit(&bars->o_done[1], lead);
                    if (j > 0) commit(&bars->v_empty[(j - 1) & 1], lead);
                    if (next1) qk(1, j, next1);
                    if (j < w.n) commit(&bars->k_empty[j & 1], lead);
                    keys0 = next0;
                    keys1 = next1;
                    if (__any_sync(0xffffffffu, !ok)) break;
                    if (j >= whole0 && j + 1 < whole1) {
#pragma unroll 1
                        while (j + 1 < whole1 && !__any_sync(0xffffffffu, !ok)) {
                            ++j;
                            if (j & 1) whole_step(std::integral_constant<int, 1>{}, (uint32_t)(j >> 1) & 1u, (uint32_t)((j - 1) >> 1) & 1u);
                            else whole_step(std::integral_constant<int, 0>{}, (uint32_t)(j >> 1) & 1u, (uint32_t)((j - 1) >> 1) & 1u);
                        }
                    }
                }
                // After a wait that gave up the tensor pipe still drains before TMEM is freed.
                if (j < w.n) {
                    commit(&bars->o_done[0], lead);
                    commit(&bars->o_done[1], lead);
                }
            }
        } else if (warp == 2) {
            for (int j = 0; j < w.n; ++j) {
                const int st = j & 1;
                if (!__all_sync(0xffffffffu, sm100::mbar_wait(&bars->v_full[st], (uint32_t)(j >> 1) & 1u, status, 126))) break;
                const int rows = (max(span0.count(w, j), span1.count(w, j)) + 15) & ~15;
                const int real = min(rows, ke - kb - w.start(j));
                for (int i = lane; i < DB * (rows - real) * 8; i += 32) {
                    const int b = i / ((rows - real) * 8), rest = i % ((rows - real) * 8);
                    *reinterpret_cast<uint4*>(smem + L::V + st * L::TILE + b * BOX + (real + rest / 8) * 128 + (rest % 8) * 16) = make_uint4(0, 0, 0, 0);
                }
                if (real < rows) sm100::fence_proxy_async_smem();
                sm100::mbar_arrive(&bars->v_ready[st]);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        const int t = (warp >> 2) - 1;
        const int row = (warp & 3) * 32 + lane;
        const int tok = row / a.group;
        const int n_tok = t ? rows_tok[1] : rows_tok[0];
        const Span span = t ? span1 : span0;
        const int first = span.first;
        const bool live = row < qrows && tok < n_tok;
        const int p = live ? first + tok : -1;
        const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + 128u * t + lane_off, to = tmem + O_COL + 128u * t + lane_off;
        RowState s{-INFINITY, 0.f};
        uint32_t turn = 0;
        bool ok = true;
        for (int j = 0; j < w.n; ++j) {
            if (!span.active(w, j)) continue;
            if (!wait_soon(&bars->s_full[t], turn & 1u, status, 127)) {
                ok = false;
                break;
            }
            sm100::tc_fence_after();
            float2 acc[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
            uint32_t r[128];
            if (span.full(w, j, a.sinks)) {
#pragma unroll
                for (int c = 0; c < 4; ++c) sm100::tmem_ld_32x32b_x32(ts + 32u * c, *reinterpret_cast<uint32_t(*)[32]>(&r[32 * c]));
                sm100::tmem_ld_wait();
                float mx = -INFINITY;
#pragma unroll
                for (int c = 0; c < 4; ++c) mx = max32(r + 32 * c, mx);
                const float m = s.raise<T, D>(mx, a.scale_log2, to, turn > 0);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t pw[32];
                    weights32<T>(r + 32 * c, a.scale_log2, m, acc, pw);
                    sm100::tmem_st_32x32b_x32(ts + 32u * c, pw);
                    if (c == FIRST_KEYS / 32 - 1 || c == 3) {
                        sm100::tmem_st_wait();
                        sm100::tc_fence_before();
                        sm100::mbar_arrive(&bars->p_full[t][c == 3]);
                    }
                }
            } else {
                // 32 columns at a time, as many as the tile has.  Column c of the tile is seen when c < end
                // and (c >= begin or c < sink).
                const int chunks = (span.count(w, j) + 31) >> 5;
                const int start = w.start(j);
                const bool in_sinks = w.in_sinks(j);
                const int end = in_sinks ? (p >= 0 ? w.sink_end - start : 0) : p + 1 - start;
                const int begin = in_sinks || !a.window ? 0 : p - a.window + 1 - start;
                const int sink = a.sinks - start;
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (c < chunks) sm100::tmem_ld_32x32b_x32(ts + 32u * c, *reinterpret_cast<uint32_t(*)[32]>(&r[32 * c]));
                sm100::tmem_ld_wait();
                float mx = -INFINITY;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    if (c >= chunks) continue;
                    const uint32_t seen = below(end - 32 * c) & (~below(begin - 32 * c) | below(sink - 32 * c));
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (!(seen >> i & 1u)) r[32 * c + i] = 0xff800000u;
                    mx = max32(r + 32 * c, mx);
                }
                const float m = s.raise<T, D>(mx, a.scale_log2, to, turn > 0);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    if (c >= chunks) continue;
                    uint32_t pw[32];
                    weights32<T>(r + 32 * c, a.scale_log2, m, acc, pw);
                    sm100::tmem_st_32x32b_x32(ts + 32u * c, pw);
                }
                sm100::tmem_st_wait();
                sm100::tc_fence_before();
                sm100::mbar_arrive(&bars->p_full[t][0]);
                sm100::mbar_arrive(&bars->p_full[t][1]);
            }
            s.l += acc[0].x + acc[0].y + acc[1].x + acc[1].y;
            ++turn;
        }
        // ---- O / l ----
        // Through the tile's Q buffer (its products are done), so that 16 (8) lanes store a whole row; a
        // row's 16-byte pieces are turned by its number to spread over the banks.
        float2 nan = sf::f2(0.f);
        if (w.n > 0) ok = wait_soon(&bars->o_done[t], 0, status, 128) && ok;
        sm100::tc_fence_after();
        if (parts > 1) {
            // The row's state for the join, O as it is: half its columns at a time through the Q buffer.
            const bool own = live && ok;
            const int64_t row_at = LINE ? ((int64_t)part * rest + pair - a.whole) * (2 * qrows) + t * qrows + row
                                        : ((int64_t)part * a.tq + tok0 + t * tq_tile + tok) * a.heads + kvh * a.group + row - tok * a.group;
            if (own) *reinterpret_cast<float2*>(a.stat + 2 * row_at) = make_float2(turn ? s.m : -INFINITY, s.l);
            const uint32_t written = __ballot_sync(0xffffffffu, own);
            constexpr int PIECES = D / 8;  // 16-byte pieces of half a row
            uint4* stage = reinterpret_cast<uint4*>(smem + L::Q + t * L::TILE) + (warp & 3) * 32 * PIECES;
#pragma unroll 1
            for (int half = 0; half < 2 && turn; ++half) {
#pragma unroll 1
                for (int c = 0; c < D / 64; ++c) {
                    uint32_t r[32];
                    sm100::tmem_ld_32x32b_x32(to + (uint32_t)(half * D / 2 + 32 * c), r);
                    sm100::tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 8; ++i) stage[lane * PIECES + ((8 * c + i) ^ (lane & 7))] = make_uint4(r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]);
                }
                __syncwarp();
#pragma unroll 4
                for (int i = lane; i < 32 * PIECES; i += 32) {
                    const int rl = i / PIECES, piece = i % PIECES;
                    const int64_t at = __shfl_sync(0xffffffffu, row_at, rl);
                    const uint4 x = stage[rl * PIECES + (piece ^ (rl & 7))];
                    if (written >> rl & 1u) *reinterpret_cast<uint4*>(a.part + at * D + half * D / 2 + 4 * piece) = x;
                }
                __syncwarp();
            }
        } else {
            const bool none = turn == 0 || p < 0;
            const float inv = 1.0f / s.l;
            constexpr int PIECES = D / 8;
            uint4* stage = reinterpret_cast<uint4*>(smem + L::Q + t * L::TILE) + (warp & 3) * 32 * PIECES;
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
                uint32_t r[32];
                sm100::tmem_ld_32x32b_x32(to + 32u * c, r);
                sm100::tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t o4[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float2 x = make_float2(__uint_as_float(r[8 * i + 2 * e]) * inv, __uint_as_float(r[8 * i + 2 * e + 1]) * inv);
                        if (none) x = make_float2(0.f, 0.f);
                        nan = sf::f2_fma(x, sf::f2(0.f), nan);  // 0, or NaN once a NaN or an infinity has passed
                        o4[e] = sf::Pair<T>::from_f2(x);
                    }
                    stage[lane * PIECES + ((4 * c + i) ^ (lane & 7))] = make_uint4(o4[0], o4[1], o4[2], o4[3]);
                }
            }
            const bool again = live && ok && !(nan.x + nan.y == 0.f) && s.l < INFINITY;
            const int64_t mine = (int64_t)(tok0 + t * tq_tile + tok) * a.ot + (int64_t)(kvh * a.group + row - tok * a.group) * a.oh;
            __syncwarp();
            const uint32_t written = __ballot_sync(0xffffffffu, live && ok);
#pragma unroll 4
            for (int i = lane; i < 32 * PIECES; i += 32) {
                const int rl = i / PIECES, piece = i % PIECES;
                const int64_t at = __shfl_sync(0xffffffffu, mine, rl);
                const uint4 x = stage[rl * PIECES + (piece ^ (rl & 7))];
                if (written >> rl & 1u) *reinterpret_cast<uint4*>((T*)a.o + at + 8 * piece) = x;
            }
            __syncwarp();
            settle<T, D>(a, again, p, kb, (int64_t)tok0 + t * tq_tile + tok, kvh * a.group + row - tok * a.group, (T*)a.o + mine);
        }
    }
    sm100::tc_fence_before();
    __syncthreads();
    sm100::tc_fence_after();
    if (warp == 1) sm100::tmem_dealloc(tmem, 512);
}

// Join the splits of every row.  Tokens are found as in the kernel above; its 256 rows are dealt to blocks of
// JOIN_ROWS.  A warp takes its ROWS rows side by side, each split's state in turn onto a running max, so the
// trips to L2 overlap: 1536 tokens, 28 heads of 128 and 8200 keys in 3 parts take 206 us in all with a row at a
// time behind its max, 197 so, 198 and 200 in blocks of 32 and 64 rows.
constexpr int JOIN_ROWS = 16;
template <typename T, int D>
__global__ void __launch_bounds__(256) window_join_kernel(const __grid_constant__ Args a, int tq_tile) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    int slot = blockIdx.x, kvh = blockIdx.y;
    if (a.whole) {
        const int pair = a.whole + blockIdx.x;
        kvh = pair / a.slots;
        slot = a.slots - 1 - (pair - kvh * a.slots);
    }
    Where at;
    if (!locate(a, 2 * tq_tile, slot, &at)) return;
    constexpr int ROWS = JOIN_ROWS / 8, E = D / 32;
    const int lane = threadIdx.x & 31;
    const int r0 = blockIdx.z * JOIN_ROWS + (threadIdx.x >> 5) * ROWS;
    const int rows = max(0, min(ROWS, min(2 * tq_tile, at.qe - at.tok0) * a.group - r0));
    __shared__ uint32_t again_s;  // of the block's rows, those that have to be settled
    if (threadIdx.x == 0) again_s = 0;
    __syncthreads();
    const int64_t all = a.whole ? (int64_t)gridDim.x * (2 * tq_tile * a.group) : a.tq * a.heads;
    int64_t row_at[ROWS];
    float m[ROWS], l[ROWS], acc[ROWS][E];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int r = r0 + min(i, max(0, rows - 1)), tok = r / a.group;
        row_at[i] = a.whole ? (int64_t)blockIdx.x * (2 * tq_tile * a.group) + r : (int64_t)(at.tok0 + tok) * a.heads + kvh * a.group + r - tok * a.group;
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[i][e] = 0.f;
    }
    for (int z = 0; z < (rows ? a.splits : 0); ++z) {
        float2 st[ROWS];
        float x[ROWS][E];
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            const int64_t from = z * all + row_at[i];
            st[i] = *reinterpret_cast<const float2*>(a.stat + 2 * from);
            if constexpr (E == 4) *reinterpret_cast<float4*>(x[i]) = *reinterpret_cast<const float4*>(a.part + from * D + E * lane);
            else *reinterpret_cast<float2*>(x[i]) = *reinterpret_cast<const float2*>(a.part + from * D + E * lane);
        }
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            if (st[i].x == -INFINITY) continue;  // that split saw nothing and left no output
            const float mn = st[i].x > m[i] || st[i].x != st[i].x ? st[i].x : m[i];
            const float f = exp2f(m[i] - mn), g = exp2f(st[i].x - mn);
            m[i] = mn;
            l[i] = l[i] * f + st[i].y * g;
#pragma unroll
            for (int e = 0; e < E; ++e) acc[i][e] = acc[i][e] * f + x[i][e] * g;
        }
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        if (i >= rows) break;
        const int tok = (r0 + i) / a.group, head = kvh * a.group + r0 + i - tok * a.group, p = at.pos0 + tok;
        const float inv = 1.0f / l[i];
        bool again = false;
        T* out = (T*)a.o + (int64_t)(at.tok0 + tok) * a.ot + (int64_t)head * a.oh;
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            float2 v = make_float2(acc[i][e] * inv, acc[i][e + 1] * inv);
            if (p < 0) v = make_float2(0.f, 0.f);
            again |= !(v.x * 0.f + v.y * 0.f == 0.f);
            *reinterpret_cast<uint32_t*>(out + E * lane + e) = sf::Pair<T>::from_f2(v);
        }
        if (__any_sync(0xffffffffu, again) && l[i] < INFINITY && lane == 0) atomicOr(&again_s, 1u << (ROWS * (threadIdx.x >> 5) + i));
    }
    __syncthreads();
    if (again_s && threadIdx.x < 32) {  // one warp for the block's rows, a lane each
        const int r = blockIdx.z * JOIN_ROWS + lane, tok = r / a.group, head = kvh * a.group + r - tok * a.group;
        settle<T, D>(a, again_s >> lane & 1u, at.pos0 + tok, at.kb, (int64_t)at.tok0 + tok, head,
                     (T*)a.o + (int64_t)(at.tok0 + tok) * a.ot + (int64_t)head * a.oh);
    }
}

// CTAs that share the keys of a pair of row tiles.  A tile of 128 keys takes a CTA about 1.9 us, a CTA's start
// and end some 4, and a row's state leaves and comes back through L2: the least estimate of that over the SMs, if
// it is a twentieth below the unsplit one's.  The lengths are on the GPU, so pairs and tiles are those of sequences of
// equal length.
// bf16, 32 query heads on 8 key heads of 128, no window: 1 token x 32768 keys 514 us unsplit, 51 us at the 16
// chosen; 64 x 8192 138 and 33 (16); 64 x 32768 527 and 61 (16); 512 x 32768 544 and 306 (2).
// Where the pairs are more than a round of CTAs, those of the whole rounds keep their keys and only the last,
// partial round's are split, and only their states are in the workspace: 1536 tokens in 3 prompts behind 8200, 28
// heads on 4 (177 pairs) 317 us unsplit, 226 so, 17 MB; 1280 x 8192 (160 pairs) 279 and 199, 21 MB; not for 16384
// tokens behind 65536, where a percent would have to be gained.
struct Split {
    int64_t z, whole;
    int64_t rows;  // whose states a part leaves in the workspace
    uint64_t bytes(int64_t D) const { return z > 1 ? (uint64_t)(z * rows * (D + 2) * 4) : 0; }
};
// The states stay in L2 (126 MB) until they are joined; 1000 tokens behind 500000 would else have 32 parts and 470 MB.
constexpr double MOST_STATES = 96e6;
Split split_of(int64_t Tq, int64_t Tk, int64_t seqs, int64_t Hq, int64_t Hk, int64_t D, int64_t window, int64_t sinks) {
    const int64_t group = Hq / Hk;
    Split pick = {1, 0, 0};
    if ((D != 64 && D != 128) || group > 128 || Tk == 0 || seqs == 0) return pick;
    const int64_t tt = 2 * (128 / group), tokens = (Tq + seqs - 1) / seqs;
    const double pairs = (double)(std::min(seqs, Tq) * ((tokens + tt - 1) / tt) * Hk);
    // Key tiles of a pair: of the first tokens, which see the fewest, and on average (keys from a to b, at most w each).
    const double b = (double)Tk / seqs, a = std::max(1.0, b - tokens);
    const double w = window ? std::min(b, (double)window + tt + std::min<double>((double)sinks, b)) : b;
    const double few = std::min(a, w) / 128 + 0.5, mean = (b <= w || a >= w ? (std::min(a, w) + std::min(b, w)) / 2 : ((w * w - a * a) / 2 + w * (b - w)) / (b - a)) / 128 + 0.5;
    const double sms = sf::sm_count(), rounds = std::floor(pairs / sms), rest = pairs - rounds * sms;
    constexpr double ENDS = 2.2;  // a CTA's start and end, in tiles; so is the join's launch
    // n CTAs of `tiles` tiles on average, the heaviest first: their sum over the SMs, and what the last round leaves idle.
    auto time = [&](double n, double tiles, double least) { return n * (tiles + ENDS) / sms + (std::ceil(n / sms) - n / sms) * (least + ENDS); };
    // Of the pairs in the grid, those of the whole rounds; the slots that rounding leaves over lie among the others.
    const double slots = (double)(Tq / tt + seqs) * Hk, whole = std::floor(rounds * sms * slots / pairs), split = slots - whole;
    double best = 0.95 * time(pairs, mean, few);
    for (int64_t z : {2, 3, 4, 6, 8, 12, 16, 24, 32}) {
        if (mean < 2 * z) break;
        const double join = (double)Tq * Hq * D * 8 * z / 12e6;  // 12 MB of states in a tile's time
        const double all = time(pairs * z, mean / z, few / z) + ENDS + join;
        const double last = rounds * (mean + ENDS) + time(rest * z, mean / z, few / z) + 1.7 * ENDS + join * rest / pairs;
        auto fits = [&](double rows) { return z * rows * (D + 2) * 4 <= MOST_STATES; };
        if (all < best && fits((double)Tq * Hq)) best = all, pick = {z, 0, Tq * Hq};
        if (rounds > 0 && rest > 0 && split > 0 && last < best && whole + split * z <= 0x7fffffff && fits(split * tt * group))
            best = last, pick = {z, (int64_t)whole, (int64_t)split * tt * group};
    }
    return pick;
}

// Whether the tensor-core kernel takes these tensors; `rows` token and head strides of an [n, h, D] tensor.
bool tc_rows(const void* p, int64_t token, int64_t head, int64_t n, int64_t h) {
    return sf::aligned16(p) && (n <= 1 || (token > 0 && token % 8 == 0)) && (h <= 1 || (head > 0 && head % 8 == 0));
}

template <typename T, int D>
int launch_tc(Args a, int64_t hk, bool* taken, cudaStream_t st, char* err, uint64_t cap) {
    const bool bf16 = std::is_same<T, __nv_bfloat16>::value;
    const int tq_tile = 128 / a.group;
    auto map = [&](CUtensorMap* m, const void* p, int64_t token, int64_t head, int64_t n, int64_t h, int bh, int bn) {
        return sf::tmap_3d_encode(m, p, D, h, n, h > 1 ? head * 2 : D * 2, n > 1 ? token * 2 : D * 2, 64, bh, bn, bf16);
    };
    CUtensorMap mq, mk, mk16, mv, mv16;
    *taken = map(&mq, a.q, a.qt, a.qh, a.tq, a.heads, a.group, tq_tile) && map(&mk, a.k, a.kt, a.kh, a.tk, hk, 1, 128) &&
             map(&mk16, a.k, a.kt, a.kh, a.tk, hk, 1, 16) && map(&mv, a.v, a.vt, a.vh, a.tk, hk, 1, 128) && map(&mv16, a.v, a.vt, a.vh, a.tk, hk, 1, 16);
    if (!*taken) return SF_OK;
    constexpr int smem = Layout<D>::BYTES + 1024 > 120 * 1024 ? Layout<D>::BYTES + 1024 : 120 * 1024;  // one CTA (all of TMEM) an SM
    {
        static std::mutex mu;
        static uint64_t done = 0;
        int dev = 0;
        cudaGetDevice(&dev);
        std::lock_guard<std::mutex> lock(mu);
        if (dev >= 64 || !(done >> dev & 1)) {
            cudaError_t e = cudaFuncSetAttribute(window_tc_kernel<T, D, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
            if (e == cudaSuccess) e = cudaFuncSetAttribute(window_tc_kernel<T, D, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
            if (e != cudaSuccess) return sf::fail(SF_EDEVICE, err, cap, "window_attention: %s", cudaGetErrorString(e));
            if (dev < 64) done |= 1ull << dev;
        }
    }
    const int64_t slots = a.tq / (2 * tq_tile) + a.seqs;
    if (slots > 0x7fffffffLL) return sf::fail(SF_EINVAL, err, cap, "window_attention: grid too large");
    a.slots = (int)slots;
    const int64_t rest = slots * hk - a.whole;  // pairs of row tiles that are split
    const auto kernel = a.whole ? window_tc_kernel<T, D, true> : window_tc_kernel<T, D, false>;
    const dim3 grid = a.whole ? dim3((unsigned)(a.whole + rest * a.splits)) : dim3((unsigned)slots, (unsigned)hk, (unsigned)a.splits);
    kernel<<<grid, TC_THREADS, smem, st>>>(a, mq, mk, mk16, mv, mv16, tq_tile);
    int rc = sf::check_launch("window_attention launch", err, cap);
    if (rc || a.splits == 1) return rc;
    cudaLaunchConfig_t cfg = {};
    const unsigned blocks = (unsigned)((2 * tq_tile * a.group + JOIN_ROWS - 1) / JOIN_ROWS);
    cfg.gridDim = a.whole ? dim3((unsigned)rest, 1, blocks) : dim3((unsigned)slots, (unsigned)hk, blocks);
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, window_join_kernel<T, D>, (const Args)a, (int)tq_tile);
    if (e != cudaSuccess) return sf::fail(SF_EDEVICE, err, cap, "window_attention join launch: %s", cudaGetErrorString(e));
    return SF_OK;
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

extern "C" uint64_t sf_window_attention_workspace_bytes(int64_t Tq, int64_t Tk, int64_t seqs, int64_t Hq, int64_t Hk, int64_t D, int64_t window,
                                                        int64_t sinks) {
    if (Tq <= 0 || Tk <= 0 || seqs <= 0 || Hq <= 0 || Hk <= 0 || Hq % Hk || window < 0 || sinks < 0) return 0;
    return split_of(Tq, Tk, seqs, Hq, Hk, D, window < Tk ? window : 0, sinks).bytes(D);
}

extern "C" int sf_window_attention(const sf_window_attention_args* x, void* stream, char* err, uint64_t cap) {
    if (!x) return sf::fail(SF_EINVAL, err, cap, "window_attention: null arguments");
    const int64_t Tq = x->Tq, Tk = x->Tk, seqs = x->seqs, Hq = x->Hq, Hk = x->Hk, D = x->D;
    const float scale = (float)x->scale;
    if (Tq < 0 || Tk < 0 || seqs < 0 || Hq < 0 || Hk < 0 || D < 1) return sf::fail(SF_EINVAL, err, cap, "window_attention: bad sizes");
    if (Hq && (Hk == 0 || Hq % Hk)) return sf::fail(SF_EINVAL, err, cap, "window_attention: the query heads must be a multiple of the key heads");
    if (Tq > 0x7fffffffLL || Tk > 0x7fffffffLL || seqs > 0x7fffffffLL || Hq > (1 << 20))
        return sf::fail(SF_EINVAL, err, cap, "window_attention: size above 2^31 - 1");
    if (!(scale > 0.f) || !(scale < INFINITY)) return sf::fail(SF_EINVAL, err, cap, "window_attention: scale must be > 0");
    if (x->variant != 0 && x->variant != 1 && x->variant != 2 && x->variant != 4)
        return sf::fail(SF_EINVAL, err, cap, "window_attention: no variant %d", x->variant);
    if (x->window < 0 || x->sinks < 0) return sf::fail(SF_EINVAL, err, cap, "window_attention: window and sinks must be >= 0");
    if (x->dtype != SF_DTYPE_F16 && x->dtype != SF_DTYPE_BF16) return sf::fail(SF_EINVAL, err, cap, "window_attention: dtype %d is not fp16/bf16", x->dtype);
    for (const sf_rows* r : {&x->q_rows, &x->k_rows, &x->v_rows, &x->o_rows})
        if (r->token < 0 || r->head < 0) return sf::fail(SF_EINVAL, err, cap, "window_attention: negative stride");
    if (Tq * Hq == 0 || seqs == 0) return SF_OK;
    if (!x->q || !x->o || !x->cu_q || !x->cu_k || (Tk && (!x->k || !x->v))) return sf::fail(SF_EINVAL, err, cap, "window_attention: null tensor pointer");
    Args a = {};
    a.q = x->q, a.k = x->k, a.v = x->v, a.o = x->o;
    a.cu_q = (const int32_t*)x->cu_q, a.cu_k = (const int32_t*)x->cu_k;
    a.qt = x->q_rows.token, a.qh = x->q_rows.head, a.kt = x->k_rows.token, a.kh = x->k_rows.head;
    a.vt = x->v_rows.token, a.vh = x->v_rows.head, a.ot = x->o_rows.token, a.oh = x->o_rows.head;
    a.tq = Tq, a.tk = Tk;
    a.seqs = (int)seqs, a.group = (int)(Hq / Hk), a.heads = (int)Hq;
    // Positions are below Tk, so a window of Tk keys leaves none out: below, position - window stays within 32 bits.
    const int64_t window = x->window < Tk ? x->window : 0;
    a.window = (int)window;
    a.sinks = window ? (int)std::min<int64_t>(x->sinks, 0x7fffffff) : 0;
    a.scale_log2 = scale * LOG2E;
    a.splits = 1;
    if (x->variant != 4) {
        const Split split = split_of(Tq, Tk, seqs, Hq, Hk, D, window, x->sinks);
        if (split.z > 1 && x->workspace && sf::aligned16(x->workspace) && x->workspace_bytes >= split.bytes(D)) {
            a.splits = (int)split.z;
            a.whole = (int)split.whole;
            a.part = (float*)x->workspace;
            a.stat = a.part + split.z * split.rows * D;
        }
    }
    cudaStream_t st = (cudaStream_t)stream;
    const bool half = x->dtype == SF_DTYPE_F16;
    const bool tc = (D == 64 || D == 128) && a.group <= 128 && Hk <= 65535 && Tk > 0 && tc_rows(a.q, a.qt, a.qh, Tq, Hq) && tc_rows(a.k, a.kt, a.kh, Tk, Hk) &&
                    tc_rows(a.v, a.vt, a.vh, Tk, Hk) && tc_rows(a.o, a.ot, a.oh, Tq, Hq);
    if (x->variant == 1 && !tc)
        return sf::fail(SF_EINVAL, err, cap, "window_attention: the tensor-core variant needs D 64 or 128, at most 128 query heads a key head, 16-byte aligned tensors and strides");
    if (tc && x->variant != 2) {
        bool taken = false;
        const int rc = D == 64 ? (half ? launch_tc<__half, 64>(a, Hk, &taken, st, err, cap) : launch_tc<__nv_bfloat16, 64>(a, Hk, &taken, st, err, cap))
                               : (half ? launch_tc<__half, 128>(a, Hk, &taken, st, err, cap) : launch_tc<__nv_bfloat16, 128>(a, Hk, &taken, st, err, cap));
        if (rc || taken) return rc;
        if (x->variant == 1) return sf::fail(SF_EDEVICE, err, cap, "window_attention: the driver refused a tensor map");
    }
    if (half) return launch_general<__half>(a, D, st, err, cap);
    return launch_general<__nv_bfloat16>(a, D, st, err, cap);
}

int sf_window_status_read(uint32_t* code, uint32_t* where, cudaStream_t stream) {
    sm100::KernelStatus h{0, 0};
    if (cudaMemcpyFromSymbolAsync(&h, g_window_status, sizeof(h), 0, cudaMemcpyDeviceToHost, stream) != cudaSuccess) return SF_EDEVICE;
    if (cudaStreamSynchronize(stream) != cudaSuccess) return SF_EDEVICE;
    if (h.code) {
        const sm100::KernelStatus zero{0, 0};
        cudaMemcpyToSymbolAsync(g_window_status, &zero, sizeof(zero), 0, cudaMemcpyHostToDevice, stream);
        cudaStreamSynchronize(stream);
    }
    *code = h.code;
    *where = h.where;
    return SF_OK;
}
