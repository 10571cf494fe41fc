// Single-token attention over the 4-bit paged key/value cache (format: kv4.cuh), sm_100a:
//
//   o[b, h, :] = sum_j softmax_j(scale q[b, h, :] . k_j) v_j
//   over keys j < n_b with j >= n_b - window or j < sinks (window 0: all), k, v = minimum + scale * code
//
// HBM-bound: every record (16 keys of one head, 18 D bytes) is read once for all query heads of its
// group, ~4.5 bits a value.  What has to be kept up with is turning 4-bit codes into MMA operands,
// so the scales and minima stay out of it:
//
//   q . k_j = sum_G s_jG (q_G . c_jG) + m_jG sum(q_G)          codes c are the MMA operand,
//   o       = sum_j (p_j s_jG) (c_j - 8) + p_j (m_jG + 8 s_jG)  scales go into p, which is small.
//
//  * K: an fp16 whose low bits are a code is the subnormal c 2^-24, exactly, so one AND makes two
//    operands.  q is scaled by a power of two to [1, 2) a head (exact in fp16 down to 2^-24 of the
//    head's largest) and by 16 where the code sits in the lower nibble of its byte.
//  * V: 0x4300 | c is the bf16 128 + c; taking off 136 leaves c - 8 exactly.  Centred codes keep the
//    fp32 accumulator from growing one-sided.  p s is rounded to bf16 (as flash attention rounds p);
//    for fp16 tensors it is split into two bf16 parts, 16 bits in all.
//  * S^T = K q^T and O^T = V^T p^T (mma.sync m16n8k16, keys / elements in the 16 rows, 8 query heads
//    in the columns): a group of up to 8 heads wastes no rows, the cache is the A operand straight
//    from shared memory, and p becomes the next B operand by a transposing matrix move.  tcgen05
//    would need the expanded operands written back to shared memory, several times the cache's bytes.
//  * Each warp streams its own tiles (every 8th of the CTA's) through a ring of bulk copies, one
//    record a copy; warps meet only at the end of a (request, head) to merge their softmax states.
//  * Work is dealt in 16-key tiles: the tiles of all requests and heads in one line, an equal
//    stretch for every CTA of one resident wave, whatever the lengths.  A (request, head) that
//    spans CTAs leaves partial states in the workspace, joined by a second kernel in the order of
//    the stretches (no atomics: the same call gives the same bits).
#include "kv4.cuh"

#include <algorithm>
#include <initializer_list>
#include <mutex>
#include <type_traits>

// [0] an index out of range, [1] a wait that gave up (kept apart: a wait ends early once its word is set).
__device__ sm100::KernelStatus g_kv4_attention_status[2];

namespace {

constexpr int WARPS = 8;
constexpr int THREADS = 32 * WARPS;
constexpr int MAX_SMEM = 227 * 1024;
constexpr float LOG2E = 1.4426950408889634f;

struct Args {
    const void* q;
    void* o;
    const uint8_t* cache;
    const int32_t* table;
    const int32_t* lens;
    float* part;         // [2 grid][HB heads][D] unnormalised outputs
    float* stat;         // [2 grid][HB heads][2] running max, sum
    int32_t* chain;      // [grid][2] item joined from this CTA's last stretch on, number of pieces (0: none)
    int64_t qb, qh, ob, oh, tb;  // strides in elements
    int window, sinks;
    int B, Hk, group, blocks;    // kv heads, query heads a kv head, head blocks a kv head
    int pages, tpp, width;       // pages in the cache, tiles a page, pages a table row
    float scale_log2;
    bool split;
};

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Transpose of an 8 x 8 matrix of 16-bit values held as an MMA fragment.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t bf16x2(float a, float b) { return sf::Pair<__nv_bfloat16>::from_f2(make_float2(a, b)); }
__device__ __forceinline__ uint32_t f16x2(float a, float b) { return sf::Pair<__half>::from_f2(make_float2(a, b)); }
// (128 + c) - 136 for two codes.
__device__ __forceinline__ uint32_t centred(uint32_t x) {
    const uint32_t u = (x & 0x000F000Fu) | 0x43004300u, off = 0x43084308u;
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&u), *reinterpret_cast<const __nv_bfloat162*>(&off));
    return *reinterpret_cast<const uint32_t*>(&d);
}

// The tiles a request's query sees: [0, sink_tiles) and [first, first + n - sink_tiles).
struct Seen {
    int len, low;  // keys j < len with j >= low or j < sinks
    int n, sink_tiles, first;
    __device__ __forceinline__ Seen(const Args& a, int b) {
        len = max(0, min(__ldg(a.lens + b), a.width * a.tpp * 16));
        low = a.window && len > a.window ? len - a.window : 0;
        first = low >> 4;
        sink_tiles = low == 0 ? 0 : min((a.sinks + 15) >> 4, first);
        n = len == 0 ? 0 : sink_tiles + ((len + 15) >> 4) - first;
    }
    __device__ __forceinline__ int tile(int i) const { return i < sink_tiles ? i : first + (i - sink_tiles); }
};

template <int NG, int NT>
struct Smem {
    static constexpr int D = 64 * NG;
    static constexpr int HB = 8 * NT;               // query heads of a block
    static constexpr int STAGES = 4;
    static constexpr int PAD = D + 4;               // row stride of the staged outputs
    static constexpr int RING = WARPS * STAGES * kv4::Record<NG>::BYTES;
    static constexpr int OUT = RING;                // [warp][head][PAD] fp32
    static constexpr int STAT = OUT + WARPS * HB * PAD * 4;  // [warp][head][2] fp32
    static constexpr int BARS = STAT + WARPS * HB * 8;
    static constexpr int SCAN = BARS + WARPS * STAGES * 8;   // 8 warp sums, then the prefix of tiles
    static constexpr int bytes(int B) { return SCAN + 64 + 4 * (B + 1); }
};

// Exclusive prefix of the requests' tile counts into pre[0..B] (all threads of the CTA).
__device__ __forceinline__ void scan_tiles(const Args& a, int* pre, int* sums) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int carry = 0;
    for (int base = 0; base < a.B; base += THREADS) {
        const int b = base + threadIdx.x;
        const int n = b < a.B ? Seen(a, b).n : 0;
        int inc = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += up;
        }
        if (lane == 31) sums[warp] = inc;
        __syncthreads();
        int before = carry, all = carry;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const int s = sums[w];
            if (w < warp) before += s;
            all += s;
        }
        if (b < a.B) pre[b] = before + inc - n;
        carry = all;
        __syncthreads();
    }
    if (threadIdx.x == 0) pre[a.B] = carry;
    __syncthreads();
}

template <typename T, int NG, int NT>
__global__ void __launch_bounds__(THREADS, NT == 1 ? 2 : 1) kv4_attention_kernel(const Args a) {
    using S = Smem<NG, NT>;
    using R = kv4::Record<NG>;
    constexpr int D = 64 * NG, HB = S::HB, ST = S::STAGES;
    constexpr bool SPLIT_P = std::is_same<T, __half>::value;
    extern __shared__ __align__(128) uint8_t smem[];
    float* out_s = reinterpret_cast<float*>(smem + S::OUT);
    float* stat_s = reinterpret_cast<float*>(smem + S::STAT);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::BARS);
    int* sums = reinterpret_cast<int*>(smem + S::SCAN);
    int* pre = reinterpret_cast<int*>(smem + S::SCAN + 64);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const int row = (g & 1) ? 7 - (g >> 1) : g >> 1;  // the key of MMA row g; row g + 8 holds key row + 8

    if (lane == 0) {
        for (int i = 0; i < ST; ++i) sm100::mbar_init(&bars[warp * ST + i], 1);
        sm100::fence_mbar_init();
    }
    const int per_b = a.Hk * a.blocks;
    int64_t at = 0, end = 0;  // this CTA's stretch of the line of tiles
    int64_t share = 0;
    int b = 0;
    if (a.split) {
        scan_tiles(a, pre, sums);
        const int64_t total = (int64_t)pre[a.B] * per_b;
        share = (total + gridDim.x - 1) / gridDim.x;
        if (share < WARPS) share = WARPS;  // at least a tile a warp
        at = min(total, (int64_t)blockIdx.x * share);
        end = min(total, at + share);
        if (threadIdx.x == 0) a.chain[2 * blockIdx.x + 1] = 0;
        if (at < end) {  // the request the stretch starts in: pre[b] * per_b <= at < pre[b + 1] * per_b
            int lo = 0, hi = a.B;
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if ((int64_t)pre[mid] * per_b <= at) lo = mid;
                else hi = mid;
            }
            b = lo;
        }
        // Requests that see nothing belong to no stretch.
        for (int e = blockIdx.x; e < a.B; e += gridDim.x)
            if (pre[e + 1] == pre[e])
                for (int i = threadIdx.x; i < a.Hk * a.group * D; i += THREADS)
                    ((T*)a.o)[(int64_t)e * a.ob + (int64_t)(i / D) * a.oh + i % D] = sf::Dt<T>::from_f(0.f);
    } else {
        b = blockIdx.x / per_b;
    }
    if (blockIdx.x == 0 && threadIdx.x < 32)
        for (int e = lane; e < a.B; e += 32)
            if (__ldg(a.lens + e) > a.width * a.tpp * 16) kv4::report(g_kv4_attention_status, kv4::BAD_INDEX, kv4::AT_LENGTH);
    __syncwarp();

    uint32_t used = 0;  // tiles this warp has taken from its ring (stage = used % ST)
    bool ok = true;     // a copy that never lands ends the warp's work
    bool first_stretch = true;
    while (true) {
        // ---- the next (request, kv head, head block) and the part of its tiles that is this CTA's ----
        int kh, hb, i0, n, whole;
        if (a.split) {
            if (at >= end) break;
            while ((int64_t)pre[b + 1] * per_b <= at) ++b;
            const int64_t off = at - (int64_t)pre[b] * per_b;
            whole = pre[b + 1] - pre[b];
            const int item = (int)(off / whole);
            kh = item / a.blocks;
            hb = item - kh * a.blocks;
            i0 = (int)(off - (int64_t)item * whole);
            n = (int)min((int64_t)(whole - i0), end - at);
        } else {
            if (!first_stretch) break;
            const int item = blockIdx.x - b * per_b;
            kh = item / a.blocks;
            hb = item - kh * a.blocks;
            i0 = 0;
        }
        const Seen seen(a, b);
        if (!a.split) whole = n = seen.n;
        const int head0 = kh * a.group + hb * HB;          // first query head of the block
        const int heads = min(HB, a.group - hb * HB);

        // ---- the ring: record numbers of this warp's tiles, 32 at a time, and the first copies ----
        const int mine = n > warp ? (n - warp + WARPS - 1) / WARPS : 0;
        auto records = [&](int block) {  // of tiles 32 block + lane of this warp; -1: none, or no such page
            const int k = 32 * block + lane;
            if (k >= mine) return -1;
            const int tile = seen.tile(i0 + warp + WARPS * k);
            const int page = tile / a.tpp;
            const int id = __ldg(a.table + (int64_t)b * a.tb + page);
            if (id < 0 || id >= a.pages) {
                kv4::report(g_kv4_attention_status, kv4::BAD_INDEX, kv4::AT_PAGE);
                return -1;
            }
            return (id * a.Hk + kh) * a.tpp + (tile - page * a.tpp);
        };
        int rec_now = records(0), rec_next = records(1);
        auto issue = [&](int k, int rec) {  // lane 0: tile k of this warp, record `rec`, into its stage
            const uint32_t stage = (used + (uint32_t)k) % ST;
            uint64_t* bar = &bars[warp * ST + stage];
            if (rec < 0) {
                sm100::mbar_arrive(bar);
            } else {
                sm100::mbar_arrive_expect_tx(bar, R::BYTES);
                sm100::bulk_load(sm100::smem_u32(smem) + (warp * ST + stage) * R::BYTES, a.cache + (int64_t)rec * R::BYTES, R::BYTES, bar);
            }
        };
        int issued = ok ? min(mine, ST - 1) : 0;
        for (int k = 0; k < issued; ++k) {
            const int rec = __shfl_sync(0xffffffffu, rec_now, k);
            if (lane == 0) issue(k, rec);
        }

        // ---- q as the B operand: the lane's elements 64 G + 16 t + 0..15 of heads g (+ 8) ----
        uint32_t qf[NT][8 * NG];
        float fac[NT][2], qs[NT][2][NG];  // of heads 2t, 2t + 1
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int h = nt * 8 + g;
            float x[NG][16];
            float amax = 0.f, sum[NG];
#pragma unroll
            for (int G = 0; G < NG; ++G) {
                sum[G] = 0.f;
                const T* src = (const T*)a.q + (int64_t)b * a.qb + (int64_t)(head0 + h) * a.qh + 64 * G + 16 * t;
                uint4 raw[2] = {};
                if (h < heads) {
                    raw[0] = *reinterpret_cast<const uint4*>(src);
                    raw[1] = *reinterpret_cast<const uint4*>(src + 8);
                }
                const uint32_t w[8] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w, raw[1].x, raw[1].y, raw[1].z, raw[1].w};
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float2 f = sf::Pair<T>::to_f2(w[i]);
                    x[G][2 * i] = f.x;
                    x[G][2 * i + 1] = f.y;
                    amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
                    sum[G] += f.x + f.y;
                }
            }
#pragma unroll
            for (int o = 1; o <= 2; o <<= 1) {
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
#pragma unroll
                for (int G = 0; G < NG; ++G) sum[G] += __shfl_xor_sync(0xffffffffu, sum[G], o);
            }
            // amax 2^(137 - ex) in [2^10, 2^11): times 16 it is still an fp16.
            const uint32_t ex = min(max(__float_as_uint(amax) >> 23, 10u), 244u);
            const float up = __uint_as_float((264u - ex) << 23);
#pragma unroll
            for (int G = 0; G < NG; ++G)
#pragma unroll
                for (int h2 = 0; h2 < 2; ++h2) {
                    const float* e = &x[G][8 * h2];
                    uint32_t* f = &qf[nt][(2 * G + h2) * 4];
                    f[0] = f16x2(e[0] * up * 16.f, e[4] * up * 16.f);
                    f[1] = f16x2(e[1] * up, e[5] * up);
                    f[2] = f16x2(e[2] * up * 16.f, e[6] * up * 16.f);
                    f[3] = f16x2(e[3] * up, e[7] * up);
                }
            const float down = __uint_as_float((ex + 10u) << 23) * a.scale_log2;  // 2^(ex - 137) 2^20
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                fac[nt][c] = __shfl_sync(0xffffffffu, down, 4 * (2 * t + c));
#pragma unroll
                for (int G = 0; G < NG; ++G) qs[nt][c][G] = __shfl_sync(0xffffffffu, sum[G] * a.scale_log2, 4 * (2 * t + c));
            }
        }

        float o[NT][4 * NG][4];     // O^T: row g element 64 G + 8 g + m, row g + 8 the element 4 further; heads 2t, 2t + 1
        float m[NT][2], l[NT][2], pm[NT][2][NG];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int i = 0; i < 4 * NG; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c) o[nt][i][c] = 0.f;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                m[nt][c] = -INFINITY;
                l[nt][c] = 0.f;
#pragma unroll
                for (int G = 0; G < NG; ++G) pm[nt][c][G] = 0.f;
            }
        }

        // ---- the warp's tiles ----
        for (int k = 0; k < mine; ++k) {
            if (k && (k & 31) == 0) {
                rec_now = rec_next;
                rec_next = records((k >> 5) + 1);
            }
            __syncwarp();  // every lane is done with the stage that the next copy overwrites
            if (issued < mine && ok) {
                const int rec = __shfl_sync(0xffffffffu, (issued >> 5) == (k >> 5) ? rec_now : rec_next, issued & 31);
                if (lane == 0) issue(issued, rec);
                ++issued;
            }
            const uint32_t turn = used + (uint32_t)k;
            if (!ok && k >= issued) break;  // a copy gave up: only those in flight are still waited for
            ok &= sm100::mbar_wait(&bars[warp * ST + turn % ST], (turn / ST) & 1u, g_kv4_attention_status + 1, kv4::AT_WAIT);
            ok = __all_sync(0xffffffffu, ok);
            const bool there = __shfl_sync(0xffffffffu, rec_now, k & 31) >= 0;
            if (!ok || !there) continue;
            const uint8_t* rec = smem + (warp * ST + turn % ST) * R::BYTES;

            const int key0 = seen.tile(i0 + warp + WARPS * k) * 16;
            bool v0 = true, v1 = true;  // keys `row` and `row + 8` are seen
            const bool partly = key0 + 16 > seen.len || (key0 < seen.low && key0 + 16 > a.sinks);
            if (partly) {
                const int j = key0 + row;
                v0 = j < seen.len && (j >= seen.low || j < a.sinks);
                v1 = j + 8 < seen.len && (j + 8 >= seen.low || j + 8 < a.sinks);
            }
            // (scale, minimum) of the lane's two keys.
            float ks[2][NG], km[2][NG], vs[2][NG], vm[2][NG];
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int G = 0; G < NG; ++G) {
                    const float2 kp = sf::Pair<__nv_bfloat16>::to_f2(*reinterpret_cast<const uint32_t*>(rec + R::KP + ((row + 8 * r) * NG + G) * 4));
                    const float2 vp = sf::Pair<__nv_bfloat16>::to_f2(*reinterpret_cast<const uint32_t*>(rec + R::VP + ((row + 8 * r) * NG + G) * 4));
                    ks[r][G] = kp.x;
                    km[r][G] = kp.y;
                    const bool v = r ? v1 : v0;
                    vs[r][G] = v ? vp.x : 0.f;
                    vm[r][G] = v ? fmaf(8.f, vp.x, vp.y) : 0.f;
                }
            // S^T = K q^T, a group at a time.
            float s[NT][4];
            uint32_t kw[2][2 * NG];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const uint8_t* p = rec + R::K + (row + 8 * r) * R::ROW + t * 8 * NG;
#pragma unroll
                for (int i = 0; i < NG; ++i) {
                    if constexpr (NG == 2) {
                        if (i == 0) {
                            const uint4 w = *reinterpret_cast<const uint4*>(p);
                            kw[r][0] = w.x, kw[r][1] = w.y, kw[r][2] = w.z, kw[r][3] = w.w;
                        }
                    } else {
                        const uint2 w = *reinterpret_cast<const uint2*>(p);
                        kw[r][0] = w.x, kw[r][1] = w.y;
                    }
                }
            }
#pragma unroll
            for (int G = 0; G < NG; ++G) {
                float acc[NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) acc[nt][0] = acc[nt][1] = acc[nt][2] = acc[nt][3] = 0.f;
#pragma unroll
                for (int h2 = 0; h2 < 2; ++h2) {
                    const uint32_t x = kw[0][2 * G + h2], y = kw[1][2 * G + h2];
                    const uint32_t a0[4] = {x & 0x000F000Fu, y & 0x000F000Fu, x & 0x00F000F0u, y & 0x00F000F0u};
                    const uint32_t a1[4] = {(x >> 8) & 0x000F000Fu, (y >> 8) & 0x000F000Fu, (x >> 8) & 0x00F000F0u, (y >> 8) & 0x00F000F0u};
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const uint32_t* f = &qf[nt][(2 * G + h2) * 4];
                        mma_f16(acc[nt], a0, f[0], f[1]);
                        mma_f16(acc[nt], a1, f[2], f[3]);
                    }
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const int r = c >> 1, h = c & 1;
                        const float dot = acc[nt][c] * ks[r][G];
                        const float low = km[r][G] * qs[nt][h][G];
                        const float v = fmaf(dot, fac[nt][h], low);
                        s[nt][c] = G == 0 ? v : s[nt][c] + v;
                    }
            }
            if (partly) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    if (!v0) s[nt][0] = s[nt][1] = -INFINITY;
                    if (!v1) s[nt][2] = s[nt][3] = -INFINITY;
                }
            }
            // The running max follows only when a score passes it by 2^8: p stays within fp32 and
            // bf16 range and the final division takes the stale max out again.
            bool grow = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int h = 0; h < 2; ++h) grow |= fmaxf(s[nt][h], s[nt][h + 2]) > m[nt][h] + 8.f;
            if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float mx = fmaxf(s[nt][h], s[nt][h + 2]);
#pragma unroll
                        for (int off = 4; off < 32; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
                        mx = fmaxf(mx, m[nt][h]);
                        const float f = m[nt][h] == mx ? 1.f : exp2f(m[nt][h] - mx);
                        m[nt][h] = mx;
                        l[nt][h] *= f;
#pragma unroll
                        for (int G = 0; G < NG; ++G) pm[nt][h][G] *= f;
#pragma unroll
                        for (int i = 0; i < 4 * NG; ++i) {
                            o[nt][i][h] *= f;
                            o[nt][i][h + 2] *= f;
                        }
                    }
            }
            // p, its sum, and p s as the B operand of O^T = V^T p^T.
            uint32_t pf[NT][NG][2], pl[NT][NG][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float p[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const float mm = m[nt][c & 1];
                    p[c] = sf::ex2_ftz(s[nt][c] - (mm == -INFINITY ? 0.f : mm));
                }
                l[nt][0] += p[0] + p[2];
                l[nt][1] += p[1] + p[3];
#pragma unroll
                for (int G = 0; G < NG; ++G) {
                    pm[nt][0][G] = fmaf(p[0], vm[0][G], fmaf(p[2], vm[1][G], pm[nt][0][G]));
                    pm[nt][1][G] = fmaf(p[1], vm[0][G], fmaf(p[3], vm[1][G], pm[nt][1][G]));
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const float w0 = p[2 * r] * vs[r][G], w1 = p[2 * r + 1] * vs[r][G];
                        const uint32_t hi = bf16x2(w0, w1);
                        pf[nt][G][r] = transpose8(hi);
                        if (SPLIT_P) {
                            const float2 back = sf::Pair<__nv_bfloat16>::to_f2(hi);
                            pl[nt][G][r] = transpose8(bf16x2(w0 - back.x, w1 - back.y));
                        }
                    }
                }
            }
            // O^T += V^T p^T: the lane reads its 8 elements a group of keys t, 7 - t, 8 + t, 15 - t.
            uint32_t vw[4][NG];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int key = (i & 1 ? 7 - t : t) + 8 * (i >> 1);
                const uint8_t* p = rec + R::V + key * R::ROW + (g ^ (4 * ((key >> 1) & 1))) * 4 * NG;
                if constexpr (NG == 2) {
                    const uint2 w = *reinterpret_cast<const uint2*>(p);
                    vw[i][0] = w.x, vw[i][1] = w.y;
                } else {
                    vw[i][0] = *reinterpret_cast<const uint32_t*>(p);
                }
            }
#pragma unroll
            for (int G = 0; G < NG; ++G) {
                // Codes 0..3 and 4..7 of two keys side by side in the halves of a word.
                const uint32_t x0 = __byte_perm(vw[0][G], vw[1][G], 0x5410), x1 = __byte_perm(vw[0][G], vw[1][G], 0x7632);
                const uint32_t y0 = __byte_perm(vw[2][G], vw[3][G], 0x5410), y1 = __byte_perm(vw[2][G], vw[3][G], 0x7632);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t af[4] = {centred(x0 >> (4 * i)), centred(x1 >> (4 * i)), centred(y0 >> (4 * i)), centred(y1 >> (4 * i))};
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        mma_bf16(o[nt][4 * G + i], af, pf[nt][G][0], pf[nt][G][1]);
                        if (SPLIT_P) mma_bf16(o[nt][4 * G + i], af, pl[nt][G][0], pl[nt][G][1]);
                    }
                }
            }
        }
        used += (uint32_t)issued;  // = mine, unless a copy gave up

        // ---- the warps' states side by side, then one sum over them ----
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float sum = l[nt][h], add[NG];
#pragma unroll
                for (int G = 0; G < NG; ++G) add[G] = pm[nt][h][G];
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) {
                    sum += __shfl_xor_sync(0xffffffffu, sum, off);
#pragma unroll
                    for (int G = 0; G < NG; ++G) add[G] += __shfl_xor_sync(0xffffffffu, add[G], off);
                }
                const int head = nt * 8 + 2 * t + h;
                if (g == 0) {
                    stat_s[(warp * HB + head) * 2] = m[nt][h];
                    stat_s[(warp * HB + head) * 2 + 1] = sum;
                }
                float* dst = out_s + (warp * HB + head) * S::PAD + 8 * g;
#pragma unroll
                for (int G = 0; G < NG; ++G) {
                    *reinterpret_cast<float4*>(dst + 64 * G) =
                        make_float4(o[nt][4 * G][h] + add[G], o[nt][4 * G + 1][h] + add[G], o[nt][4 * G + 2][h] + add[G], o[nt][4 * G + 3][h] + add[G]);
                    *reinterpret_cast<float4*>(dst + 64 * G + 4) = make_float4(o[nt][4 * G][h + 2] + add[G], o[nt][4 * G + 1][h + 2] + add[G],
                                                                               o[nt][4 * G + 2][h + 2] + add[G], o[nt][4 * G + 3][h + 2] + add[G]);
                }
            }
        __syncthreads();
        const bool all_mine = n == whole;
        const int slot = 2 * blockIdx.x + (first_stretch && i0 > 0 ? 0 : 1);
        const int active = min(n, WARPS);  // warps that had tiles
        for (int e = threadIdx.x; e < HB * (D / 4); e += THREADS) {
            const int head = e / (D / 4), d = 4 * (e % (D / 4));
            float mx = -INFINITY;
            for (int w = 0; w < active; ++w) mx = fmaxf(mx, stat_s[(w * HB + head) * 2]);
            float sum = 0.f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int w = 0; w < active; ++w) {
                const float mw = stat_s[(w * HB + head) * 2];
                const float f = mw == -INFINITY && mx != -INFINITY ? 0.f : (mw == mx ? 1.f : exp2f(mw - mx));
                const float4 x = *reinterpret_cast<const float4*>(out_s + (w * HB + head) * S::PAD + d);
                sum = fmaf(f, stat_s[(w * HB + head) * 2 + 1], sum);
                acc.x = fmaf(f, x.x, acc.x);
                acc.y = fmaf(f, x.y, acc.y);
                acc.z = fmaf(f, x.z, acc.z);
                acc.w = fmaf(f, x.w, acc.w);
            }
            if (all_mine) {
                if (head < heads) {
                    const float inv = n == 0 ? 0.f : 1.0f / sum;
                    T* dst = (T*)a.o + (int64_t)b * a.ob + (int64_t)(head0 + head) * a.oh + d;
                    *reinterpret_cast<uint2*>(dst) = make_uint2(sf::Pair<T>::from_f2(make_float2(acc.x * inv, acc.y * inv)),
                                                                sf::Pair<T>::from_f2(make_float2(acc.z * inv, acc.w * inv)));
                }
            } else {
                *reinterpret_cast<float4*>(a.part + ((int64_t)slot * HB + head) * D + d) = acc;
                if (d == 0) *reinterpret_cast<float2*>(a.stat + ((int64_t)slot * HB + head) * 2) = make_float2(mx, sum);
            }
        }
        if (a.split) {
            // An item that starts here and goes on in the CTAs behind is joined from here.
            if (threadIdx.x == 0 && i0 == 0 && n < whole) {
                a.chain[2 * blockIdx.x] = b * per_b + kh * a.blocks + hb;
                a.chain[2 * blockIdx.x + 1] = (int)((at + whole - 1) / share) - blockIdx.x + 1;
            }
            at += n;
        }
        first_stretch = false;
        __syncthreads();
    }
}

// Join the pieces of the items that span CTAs: one block a (first CTA, head), 4 warps over the pieces.
template <typename T, int D, int HB>
__global__ void __launch_bounds__(128) kv4_join_kernel(const Args a) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int first = blockIdx.x, head = blockIdx.y;
    const int pieces = a.chain[2 * first + 1];
    if (pieces == 0) return;
    const int item = a.chain[2 * first];
    const int per_b = a.Hk * a.blocks;
    const int b = item / per_b, kh = (item - b * per_b) / a.blocks, hb = item - b * per_b - kh * a.blocks;
    if (hb * HB + head >= a.group) return;
    __shared__ float acc_s[4][D];
    __shared__ float stat_s[4][2];
    constexpr int E = D / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float m = -INFINITY, l = 0.f, acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
    for (int p = warp; p < pieces; p += 4) {
        // The first piece is its CTA's last stretch, the others their CTAs' first.
        const int64_t slot = (int64_t)2 * (first + p) + (p == 0 ? 1 : 0);
        const float2 st = *reinterpret_cast<const float2*>(a.stat + (slot * HB + head) * 2);
        const float* src = a.part + (slot * HB + head) * D + E * lane;
        float x[E];
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = src[e];
        const float mx = fmaxf(m, st.x);
        const float f0 = m == mx ? 1.f : exp2f(m - mx), f1 = st.x == mx ? 1.f : exp2f(st.x - mx);
        l = l * f0 + st.y * f1;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = acc[e] * f0 + x[e] * f1;
        m = mx;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) acc_s[warp][E * lane + e] = acc[e];
    if (lane == 0) {
        stat_s[warp][0] = m;
        stat_s[warp][1] = l;
    }
    __syncthreads();
    if (threadIdx.x >= D) return;
    float mx = -INFINITY, sum = 0.f, out = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) mx = fmaxf(mx, stat_s[w][0]);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        if (w >= pieces) break;
        const float f = stat_s[w][0] == mx ? 1.f : exp2f(stat_s[w][0] - mx);
        sum += f * stat_s[w][1];
        out += f * acc_s[w][threadIdx.x];
    }
    ((T*)a.o)[(int64_t)b * a.ob + (int64_t)(kh * a.group + hb * HB + head) * a.oh + threadIdx.x] = sf::Dt<T>::from_f(out / sum);
}

// Most tiles a request can see, from the table's width, window and sinks alone.
int64_t most_tiles(int64_t width, int64_t tpp, int64_t window, int64_t sinks) {
    const int64_t all = width * tpp;
    if (!window) return all;
    return std::min(all, (window + 15) / 16 + 1 + (sinks + 15) / 16);
}

struct Plan {
    int nt, blocks;
    bool split;
    int grid;
};

Plan plan_of(int64_t B, int64_t Hq, int64_t Hk, int64_t D, int64_t width, int64_t tpp, int64_t window, int64_t sinks, int32_t variant) {
    Plan p;
    const int64_t group = Hq / Hk;
    p.nt = group > 8 ? 2 : 1;
    p.blocks = (int)((group + 8 * p.nt - 1) / (8 * p.nt));
    const int64_t items = B * Hk * p.blocks;
    const int64_t wave = (int64_t)sf::sm_count() * (p.nt == 1 ? 2 : 1);
    const int64_t tiles = most_tiles(width, tpp, window, sinks);
    // Whole items a CTA while an item is at most two tiles a warp: nothing to join, no second
    // launch.  Longer items are cut so that every CTA gets the same number of tiles.
    p.split = tiles > 2 * WARPS;
    if (variant == 3) p.split = false;
    if (variant == 1) p.split = true;
    p.grid = (int)(p.split ? std::min(wave, std::max<int64_t>(1, (items * tiles + WARPS - 1) / WARPS)) : items);
    return p;
}

uint64_t workspace_of(const Plan& p, int64_t D) {
    if (!p.split) return 0;
    const uint64_t hb = 8 * p.nt;
    return (uint64_t)p.grid * (2 * hb * D * 4 + 2 * hb * 8 + 8);
}

template <typename T, int NG, int NT>
int launch_t(Args a, const Plan& p, cudaStream_t st, char* err, uint64_t cap) {
    using S = Smem<NG, NT>;
    constexpr int HB = S::HB;
    const int smem = S::bytes(p.split ? a.B : 0);
    if (smem > MAX_SMEM) return sf::fail(SF_EINVAL, err, cap, "kv4_attention: %d requests do not fit in shared memory", a.B);
    {
        static std::mutex mu;
        static uint64_t done = 0;
        int dev = 0;
        cudaGetDevice(&dev);
        std::lock_guard<std::mutex> lock(mu);
        if (dev >= 64 || !(done >> dev & 1)) {
            const cudaError_t e = cudaFuncSetAttribute(kv4_attention_kernel<T, NG, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_SMEM);
            if (e != cudaSuccess) return sf::fail(SF_EDEVICE, err, cap, "kv4_attention: %s", cudaGetErrorString(e));
            if (dev < 64) done |= 1ull << dev;
        }
    }
    kv4_attention_kernel<T, NG, NT><<<p.grid, THREADS, smem, st>>>(a);
    int rc = sf::check_launch("kv4_attention launch", err, cap);
    if (rc || !p.split) return rc;
    // The join starts while the last CTAs of the first kernel run, and waits for all of it.
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)p.grid, (unsigned)std::min(HB, a.group));
    cfg.blockDim = dim3(128);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kv4_join_kernel<T, 64 * NG, HB>, (const Args)a);
    if (e != cudaSuccess) return sf::fail(SF_EDEVICE, err, cap, "kv4_attention join launch: %s", cudaGetErrorString(e));
    return SF_OK;
}

}  // namespace

int sf_kv4_attention_status_read(uint32_t* code, uint32_t* where, cudaStream_t stream) {
    return kv4::read_status(g_kv4_attention_status, code, where, stream);
}

extern "C" uint64_t sf_kv4_attention_workspace_bytes(int64_t B, int64_t Hq, int64_t Hk, int64_t D, int64_t page_size, int64_t width, int64_t window,
                                                     int64_t sinks, int32_t variant) {
    if (B <= 0 || Hk <= 0 || Hq <= 0 || Hq % Hk || (D != 64 && D != 128) || page_size < 16 || page_size % 16 || width < 0 || window < 0 || sinks < 0) return 0;
    return workspace_of(plan_of(B, Hq, Hk, D, width, page_size / 16, window, sinks, variant), D);
}

extern "C" int sf_kv4_attention(const sf_kv4_attention_args* x, void* stream, char* err, uint64_t cap) {
    if (!x) return sf::fail(SF_EINVAL, err, cap, "kv4_attention: null arguments");
    const int64_t B = x->B, Hq = x->Hq, Hk = x->Hk, D = x->D, pages = x->pages, page_size = x->page_size, width = x->width;
    const int64_t window = x->window, sinks = x->sinks;
    const float scale = (float)x->scale;
    if (B < 0 || Hq < 0 || Hk < 0 || pages < 0 || width < 0) return sf::fail(SF_EINVAL, err, cap, "kv4_attention: negative size");
    if (D != 64 && D != 128) return sf::fail(SF_EINVAL, err, cap, "kv4_attention: D must be 64 or 128");
    if (page_size < 16 || page_size % 16) return sf::fail(SF_EINVAL, err, cap, "kv4_attention: the page size must be a multiple of 16");
    if (pages > 0x7fffffffLL / page_size || width > 0x7fffffffLL / page_size)
        return sf::fail(SF_EINVAL, err, cap, "kv4_attention: more than 2^31 - 1 slots");
    if (Hq && (Hk == 0 || Hq % Hk)) return sf::fail(SF_EINVAL, err, cap, "kv4_attention: the query heads must be a multiple of the cache's heads");
    if (!(scale > 0.f) || !(scale < INFINITY)) return sf::fail(SF_EINVAL, err, cap, "kv4_attention: scale must be > 0");
    if (window < 0 || sinks < 0) return sf::fail(SF_EINVAL, err, cap, "kv4_attention: window and sinks must be >= 0");
    if (x->dtype != SF_DTYPE_F16 && x->dtype != SF_DTYPE_BF16) return sf::fail(SF_EINVAL, err, cap, "kv4_attention: dtype %d is not fp16/bf16", x->dtype);
    for (int64_t s : {x->q_rows.token, x->q_rows.head, x->o_rows.token, x->o_rows.head})
        if (s < 0 || s % 8) return sf::fail(SF_EINVAL, err, cap, "kv4_attention: strides of q and out must be multiples of 8 elements");
    if (x->table_stride < 0) return sf::fail(SF_EINVAL, err, cap, "kv4_attention: negative table stride");
    if (B * Hq == 0) return SF_OK;
    if (!x->q || !x->o || !x->lens || (pages && !x->cache) || (width && !x->table)) return sf::fail(SF_EINVAL, err, cap, "kv4_attention: null tensor pointer");
    if (!sf::aligned16(x->q) || !sf::aligned16(x->o) || !sf::aligned16(x->cache))
        return sf::fail(SF_EINVAL, err, cap, "kv4_attention: q, out and the cache must be 16-byte aligned");
    const int64_t tpp = page_size / 16;
    if (pages * Hk > 0x7fffffffLL / tpp) return sf::fail(SF_EINVAL, err, cap, "kv4_attention: more than 2^31 - 1 records");
    // The tiles of all requests are counted in 32 bits.
    if (B > 0x7fffffffLL / std::max<int64_t>(1, width * tpp)) return sf::fail(SF_EINVAL, err, cap, "kv4_attention: requests x table width too large");
    const Plan p = plan_of(B, Hq, Hk, D, width, tpp, window, sinks, x->variant);
    if (B * Hk > 0x7fffffffLL / p.blocks) return sf::fail(SF_EINVAL, err, cap, "kv4_attention: grid too large");
    if (p.split && (!x->workspace || x->workspace_bytes < workspace_of(p, D) || !sf::aligned16(x->workspace)))
        return sf::fail(SF_EINVAL, err, cap, "kv4_attention: needs a 16-byte aligned workspace of %llu bytes", (unsigned long long)workspace_of(p, D));
    Args a = {};
    a.q = x->q;
    a.o = x->o;
    a.cache = (const uint8_t*)x->cache;
    a.table = (const int32_t*)x->table;
    a.lens = (const int32_t*)x->lens;
    if (p.split) {
        a.part = (float*)x->workspace;
        a.stat = a.part + (int64_t)p.grid * 2 * 8 * p.nt * D;
        a.chain = (int32_t*)(a.stat + (int64_t)p.grid * 2 * 8 * p.nt * 2);
    }
    a.qb = x->q_rows.token, a.qh = x->q_rows.head, a.ob = x->o_rows.token, a.oh = x->o_rows.head, a.tb = x->table_stride;
    a.window = (int)std::min<int64_t>(window, 0x7fffffff);  // lengths are below 2^31
    a.sinks = window ? (int)std::min<int64_t>(sinks, 0x7fffffff - 15) : 0;
    a.B = (int)B, a.Hk = (int)Hk, a.group = (int)(Hq / Hk), a.blocks = p.blocks;
    a.pages = (int)pages, a.tpp = (int)tpp, a.width = (int)width;
    a.scale_log2 = scale * LOG2E;
    a.split = p.split;
    const bool half = x->dtype == SF_DTYPE_F16;
    cudaStream_t st = (cudaStream_t)stream;
    if (D == 64) {
        if (p.nt == 1) return half ? launch_t<__half, 1, 1>(a, p, st, err, cap) : launch_t<__nv_bfloat16, 1, 1>(a, p, st, err, cap);
        return half ? launch_t<__half, 1, 2>(a, p, st, err, cap) : launch_t<__nv_bfloat16, 1, 2>(a, p, st, err, cap);
    }
    if (p.nt == 1) return half ? launch_t<__half, 2, 1>(a, p, st, err, cap) : launch_t<__nv_bfloat16, 2, 1>(a, p, st, err, cap);
    return half ? launch_t<__half, 2, 2>(a, p, st, err, cap) : launch_t<__nv_bfloat16, 2, 2>(a, p, st, err, cap);
}
