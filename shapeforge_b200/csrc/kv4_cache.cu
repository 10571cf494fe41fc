// Writing tokens into the 4-bit paged key/value cache and reading them back (format: kv4.cuh).
//
// HBM-bound in both directions: 4 D bytes of 16-bit values and 18 D / 16 bytes of record a token
// and head.  Four lanes hold a group of 64 elements, 16 each (two 16-byte accesses); a thread keeps
// its (head, keys or values, group, quarter) and walks the tokens, so everything but the slot is
// computed once.
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
};

// Byte offset of a slot's record for `head`.
__device__ __forceinline__ int64_t record_of(int64_t slot, int head, const Args& a, int bytes) {
    const uint32_t tile = (uint32_t)(slot >> 4);
    const uint32_t page = tile / (uint32_t)a.tiles;
    return (((int64_t)page * a.heads + head) * a.tiles + (tile - page * (uint32_t)a.tiles)) * bytes;
}

// x / s rounded as IEEE division rounds it, given y = 1 / s rounded: Markstein's final step
// (P. Markstein, "Computation of elementary functions on the IBM RISC System/6000 processor", 1990).
__device__ __forceinline__ float2 quotient(float2 x, float2 ns, float2 y) {
    const float2 q = sf::f2_mul(x, y);
    return sf::f2_fma(sf::f2_fma(q, ns, x), y, q);
}

template <typename T, int NG>
__global__ void __launch_bounds__(256) kv4_store_kernel(const Args a) {
    using R = kv4::Record<NG>;
    const Place<NG> p(a);
    const bool live = p.head < a.heads && p.token < a.per_pass;
    const T* src = live ? (const T*)(p.which ? a.v : a.k) + (int64_t)p.head * (p.which ? a.vh : a.kh) + 64 * p.group + 16 * p.quarter : nullptr;
    const int64_t ts = p.which ? a.vt : a.kt;
    for (int64_t t0 = (int64_t)blockIdx.x * a.per_pass; t0 < a.tokens; t0 += (int64_t)gridDim.x * a.per_pass) {
        const int64_t t = t0 + p.token;
        int32_t slot = live && t < a.tokens ? __ldg(a.slots + t) : -1;
        if (slot >= a.capacity) {
            kv4::report(g_kv4_status, kv4::BAD_INDEX, kv4::AT_STORE_SLOT);
            slot = -1;
        }
        uint4 raw[2] = {};
        if (slot >= 0) {
            raw[0] = *reinterpret_cast<const uint4*>(src + t * ts);
            raw[1] = *reinterpret_cast<const uint4*>(src + t * ts + 8);
        }
        float2 x[8];
        const uint32_t w[8] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w, raw[1].x, raw[1].y, raw[1].z, raw[1].w};
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
        if (slot < 0) continue;
        const float range = hi - lo;
        __nv_bfloat162 pair;
        uint32_t code[2] = {0u, 0u};
        if (range < INFINITY) {
            pair.x = __float2bfloat16_rn(range / 15.0f);
            pair.y = __float2bfloat16_rn(lo);
            const float s = __bfloat162float(pair.x), m = __bfloat162float(pair.y);
            if (s > 0.f) {
                // Both sides of the quotient times 2^64 where 1 / s would overflow.
                const float f = s < 0x1p-60f ? 0x1p64f : 1.0f;
                const float y = 1.0f / (s * f);
                const float2 ff = sf::f2(f), nm = sf::f2(-m * f), ns = sf::f2(-s * f), yy = sf::f2(y), magic = sf::f2(12582912.0f);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    // Adding 1.5 * 2^23 rounds to an integer, ties to even, in the low mantissa bits.
                    const float2 r = sf::f2_add(quotient(sf::f2_fma(x[i], ff, nm), ns, yy), magic);
                    const int c0 = __vimin_s32_relu(__float_as_int(r.x) - 0x4B400000, 15);
                    const int c1 = __vimin_s32_relu(__float_as_int(r.y) - 0x4B400000, 15);
                    code[i >> 2] |= (uint32_t)c0 << (8 * (i & 3)) | (uint32_t)c1 << (8 * (i & 3) + 4);
                }
            }
        } else {
            pair.x = __float2bfloat16_rn(0.f);
            pair.y = __float2bfloat16_rn(NAN);
        }
        const int row = slot & 15;
        uint8_t* rec = a.cache + record_of(slot, p.head, a, R::BYTES);
        if (p.which == 0) {
            *reinterpret_cast<uint2*>(rec + R::K + row * R::ROW + p.quarter * 8 * NG + p.group * 8) = make_uint2(code[0], code[1]);
        } else {
            const int c = (2 * p.quarter) ^ (4 * ((row >> 1) & 1));
            uint8_t* at = rec + R::V + row * R::ROW + p.group * 4;
            *reinterpret_cast<uint32_t*>(at + c * 4 * NG) = code[0];
            *reinterpret_cast<uint32_t*>(at + (c + 1) * 4 * NG) = code[1];
        }
        if (p.quarter == 0)
            *reinterpret_cast<uint32_t*>(rec + (p.which ? R::VP : R::KP) + (row * NG + p.group) * 4) = *reinterpret_cast<uint32_t*>(&pair);
    }
}

template <typename T, int NG>
__global__ void __launch_bounds__(256) kv4_load_kernel(const Args a) {
    using R = kv4::Record<NG>;
    const Place<NG> p(a);
    if (p.head >= a.heads || p.token >= a.per_pass) return;
    T* dst = (T*)(p.which ? a.v : a.k) + (int64_t)p.head * (p.which ? a.vh : a.kh) + 64 * p.group + 16 * p.quarter;
    const int64_t ts = p.which ? a.vt : a.kt;
    for (int64_t t = (int64_t)blockIdx.x * a.per_pass + p.token; t < a.tokens; t += (int64_t)gridDim.x * a.per_pass) {
        const int32_t slot = __ldg(a.slots + t);
        uint4 out[2] = {};
        if (slot >= 0 && slot < a.capacity) {
            const int row = slot & 15;
            const uint8_t* rec = a.cache + record_of(slot, p.head, a, R::BYTES);
            uint32_t code[2];
            if (p.which == 0) {
                const uint2 c = *reinterpret_cast<const uint2*>(rec + R::K + row * R::ROW + p.quarter * 8 * NG + p.group * 8);
                code[0] = c.x;
                code[1] = c.y;
            } else {
                const int c = (2 * p.quarter) ^ (4 * ((row >> 1) & 1));
                const uint8_t* at = rec + R::V + row * R::ROW + p.group * 4;
                code[0] = *reinterpret_cast<const uint32_t*>(at + c * 4 * NG);
                code[1] = *reinterpret_cast<const uint32_t*>(at + (c + 1) * 4 * NG);
            }
            const uint32_t pr = *reinterpret_cast<const uint32_t*>(rec + (p.which ? R::VP : R::KP) + (row * NG + p.group) * 4);
            const float2 sm = sf::Pair<__nv_bfloat16>::to_f2(pr);
            const float2 s = sf::f2(sm.x), m = sf::f2(sm.y);
            uint32_t w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t b = code[i >> 2] >> (8 * (i & 3));
                // 2^23 + q is exact, so is taking 2^23 off again.
                const float2 q = sf::f2_add(make_float2(__uint_as_float((b & 15u) | 0x4B000000u), __uint_as_float(((b >> 4) & 15u) | 0x4B000000u)),
                                            sf::f2(-8388608.0f));
                w[i] = sf::Pair<T>::from_f2(sf::f2_fma(s, q, m));
            }
            out[0] = make_uint4(w[0], w[1], w[2], w[3]);
            out[1] = make_uint4(w[4], w[5], w[6], w[7]);
        } else if (slot >= a.capacity) {
            kv4::report(g_kv4_status, kv4::BAD_INDEX, kv4::AT_LOAD_SLOT);
        }
        *reinterpret_cast<uint4*>(dst + t * ts) = out[0];
        *reinterpret_cast<uint4*>(dst + t * ts + 8) = out[1];
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
    if (x->T * x->H == 0) return SF_OK;
    if (!x->k || !x->v || !x->slots || (x->pages && !x->cache)) return sf::fail(SF_EINVAL, err, cap, "%s: null tensor pointer", what);
    if (!sf::aligned16(x->k) || !sf::aligned16(x->v) || !sf::aligned16(x->cache))
        return sf::fail(SF_EINVAL, err, cap, "%s: k, v and the cache must be 16-byte aligned", what);
    return SF_OK;
}

Args args_of(const sf_kv4_cache_args& x) {
    return Args{x.k, x.v, (const int32_t*)x.slots, (uint8_t*)x.cache, x.T, x.k_rows.token, x.k_rows.head, x.v_rows.token, x.v_rows.head,
                x.pages * x.page_size, (int)x.H, 0, (int)(x.page_size / 16)};
}

template <typename F>
int launch(F kernel, Args a, int ng, const char* what, cudaStream_t st, char* err, uint64_t cap) {
    const int lanes = 8 * ng;
    const int hc = a.heads < 256 / lanes ? a.heads : 256 / lanes;
    a.per_pass = 256 / (lanes * hc);
    const int gy = (a.heads + hc - 1) / hc;
    int64_t gx = (a.tokens + a.per_pass - 1) / a.per_pass;
    const int64_t most = (int64_t)sf::sm_count() * 16 / gy + 1;
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
        return x->D == 64 ? launch(kv4_store_kernel<__half, 1>, a, 1, "kv4_store launch", st, err, cap)
                          : launch(kv4_store_kernel<__half, 2>, a, 2, "kv4_store launch", st, err, cap);
    return x->D == 64 ? launch(kv4_store_kernel<__nv_bfloat16, 1>, a, 1, "kv4_store launch", st, err, cap)
                      : launch(kv4_store_kernel<__nv_bfloat16, 2>, a, 2, "kv4_store launch", st, err, cap);
}

extern "C" int sf_kv4_load(const sf_kv4_cache_args* x, void* stream, char* err, uint64_t cap) {
    const int rc = check("kv4_load", x, err, cap);
    if (rc || x->T * x->H == 0) return rc;
    const Args a = args_of(*x);
    cudaStream_t st = (cudaStream_t)stream;
    if (x->dtype == SF_DTYPE_F16)
        return x->D == 64 ? launch(kv4_load_kernel<__half, 1>, a, 1, "kv4_load launch", st, err, cap)
                          : launch(kv4_load_kernel<__half, 2>, a, 2, "kv4_load launch", st, err, cap);
    return x->D == 64 ? launch(kv4_load_kernel<__nv_bfloat16, 1>, a, 1, "kv4_load launch", st, err, cap)
                      : launch(kv4_load_kernel<__nv_bfloat16, 2>, a, 2, "kv4_load launch", st, err, cap);
}
