// Writing tokens into the 4-bit paged key/value cache and reading them back (format: kv4.cuh).
//
// HBM-bound in both directions: 4 D bytes of 16-bit values and 18 D / 16 bytes of record a token
// and head.  Four lanes hold a group of 64 elements, 16 each: the 16-byte pieces `quarter` and quarter
// + 4, so that a warp's accesses to the values fill whole sectors; a thread keeps its (head, keys or
// values, group, quarter) and walks the tokens, so everything but the slot is computed once.
// 32768 tokens of 8 heads of 128 in bf16: store 41 us, 4.2 TB/s, bound by its instructions (issue slots 70 % busy:
// extrema, exactly rounded quotients, packing); load 35 us, 4.9 TB/s, between DRAM and the expansion of the codes.
// Pieces that fill no whole sectors took 55 and 38 us.
#include "kv4.cuh"

#include <initializer_list>

__device__ sm100::KernelStatus g_kv4_status[2];  // [0] an index out of range; [1] unused

namespace {

struct Args {
    void* k;
    void* v;
    const int32_t* slots;
    uint8_t* cache;
    int64_t tokens, kt, kh, vt, vh;  // strides in elements
    int64_t capacity;                // slots in the cache
    int heads, per_pass, tiles;      // tokens a CTA takes at once; 16-token tiles in a page
    uint32_t magic, shift;           // n / tiles = umulhi(n, magic) >> shift for n < 2^31 (magic 0: tiles is 1)
};

// The thread's place: its share of a token, and the token it starts with.
template <int NG>
struct Place {
    int head, which, group, quarter, token;
    __device__ __forceinline__ Place(const Args& a) {
        const int lanes = 8 * NG;  // of one head: keys and values, NG groups, 4 quarters
        const int hc = min(a.heads, 256 / lanes);
        const int local = threadIdx.x % (lanes * hc);
        token = threadIdx.x / (lanes * hc);
        head = blockIdx.y * hc + local / lanes;
        which = (local / (4 * NG)) & 1;
        group = (local >> 2) % NG;
        quarter = local & 3;
    }
    // Byte in a record of the eight codes of piece quarter + 4 i in `row`.
    template <typename R>
    __device__ __forceinline__ int word(int row, int i) const {
        const int c = quarter + 4 * i;
        if (which == 0) return R::K + row * R::ROW + (c >> 1) * 8 * NG + group * 8 + (c & 1) * 4;
        return R::V + row * R::ROW + (c ^ (4 * ((row >> 1) & 1))) * 4 * NG + group * 4;
    }
};

// Byte offset of a slot's record for `head`.
__device__ __forceinline__ int64_t record_of(int32_t slot, int head, const Args& a, int bytes) {
    const uint32_t tile = (uint32_t)slot >> 4;
    const uint32_t page = a.magic ? __umulhi(tile, a.magic) >> a.shift : tile;
    return (int64_t)((page * (uint32_t)a.heads + head) * (uint32_t)a.tiles + (tile - page * (uint32_t)a.tiles)) * bytes;
}

// x / s rounded as IEEE division rounds it, given y = 1 / s rounded: Markstein's final step
// (P. Markstein, "Computation of elementary functions on the IBM RISC System/6000 processor", 1990).
__device__ __forceinline__ float2 quotient(float2 x, float2 ns, float2 y) {
    const float2 q = sf::f2_mul(x, y);
    return sf::f2_fma(sf::f2_fma(q, ns, x), y, q);
}

// Two integers saturated to 0..15 into the low byte, b in its low half, what c holds moved up by eight bits.
__device__ __forceinline__ uint32_t pack_codes(int a, int b, uint32_t c) {
    uint32_t d;
    asm("cvt.pack.sat.u4.s32.b32 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}

// A thread's 16 elements of a token, and where they go (slot < 0: nowhere).
struct Taken {
    uint4 raw[2];
    int32_t slot;
};

template <typename T, int NG>
__global__ void __launch_bounds__(256) kv4_store_kernel(const Args a) {
    using R = kv4::Record<NG>;
    const Place<NG> p(a);
    const bool live = p.head < a.heads && p.token < a.per_pass;
    const T* src = live ? (const T*)(p.which ? a.v : a.k) + (int64_t)p.head * (p.which ? a.vh : a.kh) + 64 * p.group + 8 * p.quarter : nullptr;
    const int64_t ts = p.which ? a.vt : a.kt;
    const int64_t step = (int64_t)gridDim.x * a.per_pass;
    auto take = [&](int64_t t) {
        Taken x = {};
        x.slot = live && t < a.tokens ? __ldg(a.slots + t) : -1;
        if (x.slot >= a.capacity) {
            kv4::report(g_kv4_status, kv4::BAD_INDEX, kv4::AT_STORE_SLOT);
            x.slot = -1;
        }
        if (live && t < a.tokens) {
            x.raw[0] = *reinterpret_cast<const uint4*>(src + t * ts);
            x.raw[1] = *reinterpret_cast<const uint4*>(src + t * ts + 32);
        }
        return x;
    };
    // The next token's elements are on their way while this one's are worked on.
    Taken next = take((int64_t)blockIdx.x * a.per_pass + p.token);
    for (int64_t t0 = (int64_t)blockIdx.x * a.per_pass; t0 < a.tokens; t0 += step) {
        const Taken now = next;
        next = take(t0 + step + p.token);
        float2 x[8];
        const uint32_t w[8] = {now.raw[0].x, now.raw[0].y, now.raw[0].z, now.raw[0].w, now.raw[1].x, now.raw[1].y, now.raw[1].z, now.raw[1].w};
        float lo = INFINITY, hi = -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            x[i] = sf::Pair<T>::to_f2(w[i]);
            asm("min.NaN.f32 %0, %0, %1, %2;" : "+f"(lo) : "f"(x[i].x), "f"(x[i].y));
            asm("max.NaN.f32 %0, %0, %1, %2;" : "+f"(hi) : "f"(x[i].x), "f"(x[i].y));
        }
#pragma unroll
        for (int o = 1; o <= 2; o <<= 1) {
            const float l2 = __shfl_xor_sync(0xffffffffu, lo, o), h2 = __shfl_xor_sync(0xffffffffu, hi, o);
            asm("min.NaN.f32 %0, %0, %1;" : "+f"(lo) : "f"(l2));
            asm("max.NaN.f32 %0, %0, %1;" : "+f"(hi) : "f"(h2));
        }
        if (now.slot < 0) continue;
        const float range = hi - lo;
        float s, m = __bfloat162float(__float2bfloat16_rn(lo)), y, f = 1.0f;
        if (range > 0x1p-60f && range < 0x1p100f) {
            // The quotients range / 15 and 1 / s as IEEE division rounds them: Markstein's step again for the
            // first; for the second one Newton step on the hardware's reciprocal, which rounds right for
            // every significand of 8 bits.
            s = quotient(sf::f2(range), sf::f2(-15.0f), sf::f2(1.0f / 15.0f)).x;
            s = __bfloat162float(__float2bfloat16_rn(s));
            asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(s));
            y = fmaf(y, fmaf(-s, y, 1.0f), y);
        } else if (range < INFINITY) {
            s = __bfloat162float(__float2bfloat16_rn(range / 15.0f));
            // Both sides of the quotient times 2^64 where 1 / s would overflow.
            if (s < 0x1p-60f) f = 0x1p64f;
            y = 1.0f / (s * f);
        } else {
            s = y = 0.f;
            m = NAN;
        }
        uint32_t code[2] = {0u, 0u};
        if (s > 0.f) {
            const float2 ff = sf::f2(f), nm = sf::f2(-m * f), ns = sf::f2(-s * f), yy = sf::f2(y), magic = sf::f2(12582912.0f);
#pragma unroll
            for (int i = 7; i >= 0; --i) {
                // Adding 1.5 * 2^23 rounds to an integer, ties to even, in the low mantissa bits.
                const float2 r = sf::f2_add(quotient(sf::f2_fma(x[i], ff, nm), ns, yy), magic);
                code[i >> 2] = pack_codes(__float_as_int(r.y) - 0x4B400000, __float_as_int(r.x) - 0x4B400000, code[i >> 2]);
            }
        }
        const int row = now.slot & 15;
        uint8_t* rec = a.cache + record_of(now.slot, p.head, a, R::BYTES);
        *reinterpret_cast<uint32_t*>(rec + p.template word<R>(row, 0)) = code[0];
        *reinterpret_cast<uint32_t*>(rec + p.template word<R>(row, 1)) = code[1];
        if (p.quarter == 0)
            *reinterpret_cast<uint32_t*>(rec + (p.which ? R::VP : R::KP) + (row * NG + p.group) * 4) =
                sf::Pair<__nv_bfloat16>::from_f2(make_float2(s, m));
    }
}

// Eight codes of a word to minimum + scale q.  A code left in place under 2^23's mantissa is 2^23 + 16^k q, from
// which one fma takes q exactly.
template <typename T>
__device__ __forceinline__ uint4 values(uint32_t w, float2 s, float2 m) {
    const uint32_t one = 0x4B000000u, v = w >> 20;
    auto pick = [&](uint32_t word, uint32_t mask) { return __uint_as_float((word & mask) | one); };
    const float2 q01 = sf::f2_fma(make_float2(pick(w, 0xFu), pick(w, 0xF0u)), make_float2(1.f, 0x1p-4f), make_float2(-0x1p23f, -0x1p19f));
    const float2 q23 = sf::f2_fma(make_float2(pick(w, 0xF00u), pick(w, 0xF000u)), make_float2(0x1p-8f, 0x1p-12f), make_float2(-0x1p15f, -0x1p11f));
    const float2 q45 = sf::f2_fma(make_float2(pick(w, 0xF0000u), pick(v, 0xFu)), make_float2(0x1p-16f, 1.f), make_float2(-0x1p7f, -0x1p23f));
    const float2 q67 = sf::f2_fma(make_float2(pick(v, 0xF0u), pick(v, 0xF00u)), make_float2(0x1p-4f, 0x1p-8f), make_float2(-0x1p19f, -0x1p15f));
    return make_uint4(sf::Pair<T>::from_f2(sf::f2_fma(s, q01, m)), sf::Pair<T>::from_f2(sf::f2_fma(s, q23, m)),
                      sf::Pair<T>::from_f2(sf::f2_fma(s, q45, m)), sf::Pair<T>::from_f2(sf::f2_fma(s, q67, m)));
}

template <typename T, int NG>
__global__ void __launch_bounds__(256, 6) kv4_load_kernel(const Args a) {
    using R = kv4::Record<NG>;
    const Place<NG> p(a);
    if (p.head >= a.heads || p.token >= a.per_pass) return;
    T* dst = (T*)(p.which ? a.v : a.k) + (int64_t)p.head * (p.which ? a.vh : a.kh) + 64 * p.group + 8 * p.quarter;
    const int64_t ts = p.which ? a.vt : a.kt, step = (int64_t)gridDim.x * a.per_pass;
    // Two tokens at a time: both records' reads are on their way together.
    for (int64_t t0 = (int64_t)blockIdx.x * a.per_pass + p.token; t0 < a.tokens; t0 += 2 * step) {
        int32_t slot[2];
        uint32_t code[2][2], pair[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int64_t t = t0 + u * step;
            slot[u] = t < a.tokens ? __ldg(a.slots + t) : -1;
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            code[u][0] = code[u][1] = pair[u] = 0;
            if (slot[u] >= a.capacity) {
                kv4::report(g_kv4_status, kv4::BAD_INDEX, kv4::AT_LOAD_SLOT);
                slot[u] = -1;
            }
            if (slot[u] < 0) continue;  // zeros: codes, scale and minimum
            const int row = slot[u] & 15;
            const uint8_t* rec = a.cache + record_of(slot[u], p.head, a, R::BYTES);
            code[u][0] = *reinterpret_cast<const uint32_t*>(rec + p.template word<R>(row, 0));
            code[u][1] = *reinterpret_cast<const uint32_t*>(rec + p.template word<R>(row, 1));
            pair[u] = *reinterpret_cast<const uint32_t*>(rec + (p.which ? R::VP : R::KP) + (row * NG + p.group) * 4);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int64_t t = t0 + u * step;
            if (t < a.tokens) {
                const float2 sm = sf::Pair<__nv_bfloat16>::to_f2(pair[u]);
                *reinterpret_cast<uint4*>(dst + t * ts) = values<T>(code[u][0], sf::f2(sm.x), sf::f2(sm.y));
                *reinterpret_cast<uint4*>(dst + t * ts + 32) = values<T>(code[u][1], sf::f2(sm.x), sf::f2(sm.y));
            }
        }
    }
}

int check(const char* what, const sf_kv4_cache_args* x, char* err, uint64_t cap) {
    if (!x) return sf::fail(SF_EINVAL, err, cap, "%s: null arguments", what);
    if (x->T < 0 || x->H < 0 || x->pages < 0) return sf::fail(SF_EINVAL, err, cap, "%s: negative size", what);
    if (x->D != 64 && x->D != 128) return sf::fail(SF_EINVAL, err, cap, "%s: D must be 64 or 128", what);
    if (x->page_size < 16 || x->page_size % 16) return sf::fail(SF_EINVAL, err, cap, "%s: the page size must be a multiple of 16", what);
    if (x->pages > 0x7fffffffLL / x->page_size) return sf::fail(SF_EINVAL, err, cap, "%s: the cache has more than 2^31 - 1 slots", what);
    if (x->dtype != SF_DTYPE_F16 && x->dtype != SF_DTYPE_BF16) return sf::fail(SF_EINVAL, err, cap, "%s: dtype %d is not fp16/bf16", what, x->dtype);
    if (x->H > 65535) return sf::fail(SF_EINVAL, err, cap, "%s: too many heads", what);
    for (int64_t s : {x->k_rows.token, x->k_rows.head, x->v_rows.token, x->v_rows.head})
        if (s < 0 || s % 8) return sf::fail(SF_EINVAL, err, cap, "%s: strides must be multiples of 8 elements", what);
    if (x->pages * x->H > 0x7fffffffLL / (x->page_size / 16)) return sf::fail(SF_EINVAL, err, cap, "%s: more than 2^31 - 1 records", what);
    if (x->T * x->H == 0) return SF_OK;
    if (!x->k || !x->v || !x->slots || (x->pages && !x->cache)) return sf::fail(SF_EINVAL, err, cap, "%s: null tensor pointer", what);
    if (!sf::aligned16(x->k) || !sf::aligned16(x->v) || !sf::aligned16(x->cache))
        return sf::fail(SF_EINVAL, err, cap, "%s: k, v and the cache must be 16-byte aligned", what);
    return SF_OK;
}

Args args_of(const sf_kv4_cache_args& x) {
    Args a{x.k, x.v, (const int32_t*)x.slots, (uint8_t*)x.cache, x.T, x.k_rows.token, x.k_rows.head, x.v_rows.token, x.v_rows.head,
           x.pages * x.page_size, (int)x.H, 0, (int)(x.page_size / 16), 0, 0};
    // ceil(2^(31 + s) / tiles) with 2^s >= tiles > 2^(s - 1): exact below 2^31.
    uint32_t s = 0;
    while ((1u << s) < (uint32_t)a.tiles) ++s;
    if (s) {
        a.magic = (uint32_t)(((1ull << (31 + s)) + a.tiles - 1) / (uint64_t)a.tiles);
        a.shift = s - 1;
    }
    return a;
}

template <typename F>
int launch(F kernel, Args a, int ng, int waves, const char* what, cudaStream_t st, char* err, uint64_t cap) {
    const int lanes = 8 * ng;
    const int hc = a.heads < 256 / lanes ? a.heads : 256 / lanes;
    a.per_pass = 256 / (lanes * hc);
    const int gy = (a.heads + hc - 1) / hc;
    int64_t gx = (a.tokens + a.per_pass - 1) / a.per_pass;
    const int64_t most = (int64_t)sf::sm_count() * waves / gy + 1;
    if (gx > most) gx = most;
    kernel<<<dim3((unsigned)gx, (unsigned)gy), 256, 0, st>>>(a);
    return sf::check_launch(what, err, cap);
}

}  // namespace

int sf_kv4_status_read(uint32_t* code, uint32_t* where, cudaStream_t stream) { return kv4::read_status(g_kv4_status, code, where, stream); }

extern "C" int sf_kv4_store(const sf_kv4_cache_args* x, void* stream, char* err, uint64_t cap) {
    const int rc = check("kv4_store", x, err, cap);
    if (rc || x->T * x->H == 0) return rc;
    const Args a = args_of(*x);
    cudaStream_t st = (cudaStream_t)stream;
    if (x->dtype == SF_DTYPE_F16)
        return x->D == 64 ? launch(kv4_store_kernel<__half, 1>, a, 1, 16, "kv4_store launch", st, err, cap)
                          : launch(kv4_store_kernel<__half, 2>, a, 2, 16, "kv4_store launch", st, err, cap);
    return x->D == 64 ? launch(kv4_store_kernel<__nv_bfloat16, 1>, a, 1, 16, "kv4_store launch", st, err, cap)
                      : launch(kv4_store_kernel<__nv_bfloat16, 2>, a, 2, 16, "kv4_store launch", st, err, cap);
}

extern "C" int sf_kv4_load(const sf_kv4_cache_args* x, void* stream, char* err, uint64_t cap) {
    const int rc = check("kv4_load", x, err, cap);
    if (rc || x->T * x->H == 0) return rc;
    const Args a = args_of(*x);
    cudaStream_t st = (cudaStream_t)stream;
    if (x->dtype == SF_DTYPE_F16)
        return x->D == 64 ? launch(kv4_load_kernel<__half, 1>, a, 1, 24, "kv4_load launch", st, err, cap)
                          : launch(kv4_load_kernel<__half, 2>, a, 2, 24, "kv4_load launch", st, err, cap);
    return x->D == 64 ? launch(kv4_load_kernel<__nv_bfloat16, 1>, a, 1, 24, "kv4_load launch", st, err, cap)
                      : launch(kv4_load_kernel<__nv_bfloat16, 2>, a, 2, 24, "kv4_load launch", st, err, cap);
}
