// Single-token attention over the 4-bit paged key/value cache (format: kv4.cuh), sm_100a:
//
//   o[b, h, :] = sum_j softmax_j(scale q[b, h, :] . k_j) v_j
//   over keys j < n_b with j >= n_b - window or j < sinks (window 0: all), k, v = minimum + scale * code
//
// 32 requests of up to 16384 tokens, 64 heads on 8 of 128: 80 us, 4.2 TB/s, 64 % of the floor; issue slots are 57 %
// busy with three warps a scheduler at 335 instructions a tile.  One request of 4097 tokens: 10 us, latency.
//
// HBM-bound by its bytes: every record (16 keys of one head, 18 D bytes) is read once for all query heads of its
// group, ~4.5 bits a value.  What has to be kept up with is turning 4-bit codes into MMA operands,
// so the scales and minima stay out of it:
//
//   q . k_j = sum_G s_jG (q_G . c_jG) + m_jG sum(q_G)          codes c are the MMA operand,
//   o       = sum_j (p_j s_jG) (c_j - 8) + p_j (m_jG + 8 s_jG)  scales go into p, which is small.
//
//  * K: an fp16 whose low bits are a code is the subnormal c 2^-24, exactly, so one AND makes two
//    operands.  Each head's q are scaled by a power of two of its own to at most 2^11 (an fp16 holds them
//    exactly down to 2^-25 of the head's largest; a head is a column of S^T, so nothing of it reaches another)
//    and by 16 where the code sits in the lower nibble of its byte.  The minima's part is one bf16 MMA of its
//    own: minima are bf16, sum(q_G) goes in as three bf16 parts.  S is held in units of 1024, which the
//    exponential's FMA takes out: so every finite q has a finite factor.
//  * V: with two keys' bytes side by side, 0x6400 | b is the fp16 1024 + b of a whole byte b = c + 16 c'
//    (two neighbouring elements' codes) and clearing its low bits gives 1024 + 16 c'.  Both, less 1160
//    and 1152, go through the MMA, and (c - 8) and (c' - 8) of the accumulators come from their
//    difference and a factor 1/16 at the end: two integer operations a pair of codes.  Codes taken off
//    their centre keep the fp32 accumulator from growing one-sided.  p s is an fp16 in a unit of each
//    head's own that its largest p s so far sets, so what matters of it has 11 bits (22 with the residual that
//    fp16 outputs take) whatever the values' range.
//  * S^T = K q^T and O^T = V^T p^T (mma.sync m16n8k16, keys / elements in the 16 rows, 8 query heads
//    in the columns): a group of up to 8 heads wastes no rows, the cache is the A operand straight
//    from shared memory, and p becomes the next B operand by a transposing matrix move.  tcgen05
//    would need the expanded operands written back to shared memory, several times the cache's bytes.
//  * Each warp streams its own tiles (every 4th of the CTA's) through a ring of bulk copies, one record a
//    copy; warps meet only at the end of a (request, head) to merge their softmax states.
//  * Work is dealt in 16-key tiles: the tiles of all requests and heads in one line, an equal
//    stretch for every CTA of one resident wave, whatever the lengths; each (request, head) counts
//    ITEM_COST tiles more for its start and end.  One that spans CTAs leaves partial states in the
//    workspace, joined by a second kernel in the order of the stretches (no atomics: the same call
//    gives the same bits).  A few requests of moderate length go to clusters instead, a (request, head) each:
//    one launch, its CTAs' states joined through distributed shared memory.  The first copies of a CTA's next (request, head) are issued before the
//    states of the one at hand are merged.
#include "kv4.cuh"

#include <algorithm>
#include <initializer_list>
#include <mutex>
#include <type_traits>

// [0] an index out of range, [1] a wait that gave up (kept apart: a wait ends early once its word is set).
__device__ sm100::KernelStatus g_kv4_attention_status[2];

namespace {

// Four warps a CTA and several CTAs an SM, so that one's tiles run while another starts or merges an item
// (12 warps in one CTA: 87.7 against 83.3 us for 32 requests of 8192 keys on average, 64 heads on 8); with
// one head tile (8 query heads) the registers allow a warp two key tiles side by side at a step.
constexpr int WARPS = 4;
constexpr int THREADS = 32 * WARPS;
constexpr int ctas_of(int nt) { return nt == 1 ? 3 : 2; }
constexpr int tiles_of_step(int nt) { return nt == 1 ? 2 : 1; }
constexpr int MAX_SMEM = 227 * 1024;
constexpr int LEAST = 4 * WARPS;  // tiles and costs a CTA has at least (one a warp: 13.3 against 11.6 us for one request of 4097 keys)
constexpr int ITEM_COST = 24;  // what starting and merging a (request, head) costs, in tiles
// CTAs a cluster, and tiles a CTA of one.  Against the line and its join, 32 heads on 8 of 128: one request of 1024
// tokens 7.9 and 10.2 us, 4096 10.3 and 11.6, 8192 (32 tiles a CTA) 12.8 and 13.8, 16384 (64) 18.4 and 17.5; 8
// requests of up to 2048 11.6 and 12.8, of 4096 (64 tiles a CTA) 16.7 and 14.9.
constexpr int MAX_CLUSTER = 16, CLUSTER_LEAST = 8, CLUSTER_MOST = 32;
constexpr float NO_MAX = -3e38f;  // the running max before any score
constexpr float S_UNIT = 1024.f;  // of the scores between the products and the exponential
// Smallest unit of a head's p s: p / unit stays finite for p up to 2^8.
constexpr float UNIT_FLOOR = 0x1p-118f;
// The largest p s of a head in O's unit: UNITS_NEW where it sets the unit, up to UNITS_MOST before the next does, an
// fp16 still; 2^-32 of it is a half step of the smallest.
constexpr float UNITS_NEW = 128.f, UNITS_MOST = 32768.f;
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
    bool split;                  // all tiles in a line; else `cluster` CTAs a (request, head)
    int cluster;
};

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The same onto zero.
__device__ __forceinline__ void mma_f16_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_bf16_k8_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%7,%7,%7,%7};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a0), "r"(a1), "r"(b), "f"(0.f));
}
// Transpose of an 8 x 8 matrix of 16-bit values held as an MMA fragment.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t f16x2(float a, float b) { return sf::Pair<__half>::from_f2(make_float2(a, b)); }
// a - b on two fp16.
__device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b) {
    const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&d);
}

__device__ __forceinline__ float2 ld_cluster(uint32_t at) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
    return v;
}

// The largest over the warp's keys (lanes of one t).
__device__ __forceinline__ float2 over_keys(float2 v) {
#pragma unroll
    for (int off = 4; off < 32; off <<= 1) {
        v.x = fmaxf(v.x, __shfl_xor_sync(0xffffffffu, v.x, off));
        v.y = fmaxf(v.y, __shfl_xor_sync(0xffffffffu, v.y, off));
    }
    return v;
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

// A (request, kv head, head block) and the part [i0, i0 + n) of its `whole` tiles that is this CTA's;
// n = -1: none is left.
struct Part {
    int b, item, i0, n, whole;  // item = kv head x head blocks + head block
};
// A warp's place in its CTA's stretch [at, end) of the line: the next part begins at `into` of item `item`
// of request b.  It changes once a part and would take ten registers from the loop over the tiles, so it
// is kept in shared memory, each warp its own copy.
struct Line {
    int64_t at, end;
    int b, item, into;
    Part next;
};
static_assert(sizeof(Line) <= 64, "");

template <int NG, int NT>
struct Smem {
    static constexpr int D = 64 * NG;
    static constexpr int HB = 8 * NT;               // query heads of a block
    static constexpr int TS = tiles_of_step(NT);
    static constexpr int STAGES = TS == 2 ? 3 : 4;  // steps
    static constexpr int STAGE = TS * kv4::Record<NG>::BYTES;
    static constexpr int PAD = D + 4;               // row stride of the staged outputs
    static constexpr int RING = WARPS * STAGES * STAGE;
    static constexpr int OUT = RING;                // [warp][head][PAD] fp32
    static constexpr int STAT = OUT + WARPS * HB * PAD * 4;  // [warp][head][2] fp32
    static constexpr int BARS = STAT + WARPS * HB * 8;
    static constexpr int AHEAD = BARS + (WARPS * STAGES + 2) * 8;  // [warp][64] record numbers of the next part
    static constexpr int LINE = AHEAD + WARPS * 64 * 4;            // [warp] Line
    static constexpr int SCAN = LINE + WARPS * 64;                 // prefix of the requests' costs
    static constexpr int MERGED = SCAN;                            // or, in a cluster, [head][2] fp32: the CTA's own state
    static constexpr int bytes(int B) { return SCAN + (4 * (B + 1) > HB * 8 ? 4 * (B + 1) : HB * 8); }
};

// What a request's (kv head, head block) counts in the line of tiles.
__device__ __forceinline__ int cost_of(int tiles) { return tiles ? tiles + ITEM_COST : 0; }

// Exclusive prefix of the requests' costs into pre[0..B].  Every warp computes and writes all of it (the
// same values), so none waits for another.
__device__ __forceinline__ void scan_costs(const Args& a, int* pre) {
    const int lane = threadIdx.x & 31;
    int carry = 0;
#pragma unroll 2
    for (int base = 0; base < a.B; base += 32) {
        const int b = base + lane;
        const int n = b < a.B ? cost_of(Seen(a, b).n) : 0;
        int inc = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += up;
        }
        if (b < a.B) pre[b] = carry + inc - n;
        carry += __shfl_sync(0xffffffffu, inc, 31);
    }
    if (lane == 0) pre[a.B] = carry;
    __syncwarp();
}

// JOINT: a cluster of a.cluster CTAs a (request, head), joined here.
template <typename T, int NG, int NT, bool JOINT>
__global__ void __launch_bounds__(THREADS, ctas_of(NT)) kv4_attention_kernel(const Args a) {
    using S = Smem<NG, NT>;
    using R = kv4::Record<NG>;
    constexpr int D = 64 * NG, HB = S::HB, ST = S::STAGES, TS = S::TS;
    // p s goes into its product as one fp16 for bf16 outputs, an eighth of whose step that is, and with its residual
    // for fp16 outputs.  Relative error over 32 requests of up to 16384 tokens, 64 heads on 8 of 128: bf16 1.67e-3 with
    // one part (1.66e-3 is the output's own rounding), fp16 2.9e-4 with one, 2.15e-4 with two (2.06e-4); 80 us with one
    // part, 89 with two.
    constexpr int PARTS = std::is_same<T, __half>::value ? 2 : 1;
    extern __shared__ __align__(128) uint8_t smem[];
    float* out_s = reinterpret_cast<float*>(smem + S::OUT);
    float* stat_s = reinterpret_cast<float*>(smem + S::STAT);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::BARS);
    int* pre = reinterpret_cast<int*>(smem + S::SCAN);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const int row = (g & 1) ? 7 - (g >> 1) : g >> 1;  // the key of MMA row g; row g + 8 holds key row + 8

    uint64_t* merged = bars + WARPS * ST;  // the staged states have been read (one arrival a warp)
    if (lane == 0) {
        for (int i = 0; i < ST; ++i) sm100::mbar_init(&bars[warp * ST + i], 1);
        if (warp == 0) sm100::mbar_init(merged, WARPS);
        sm100::fence_mbar_init();
    }
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the join may take its place; it waits for this grid
    const int per_b = a.Hk * a.blocks;
    Line* line = reinterpret_cast<Line*>(smem + S::LINE + 64 * warp);
    auto share_of = [&]() {  // tiles and costs a CTA
        const int64_t total = (int64_t)pre[a.B] * per_b;
        return max((int64_t)LEAST, (total + gridDim.x - 1) / gridDim.x);
    };
    if (!JOINT && a.split) {
        scan_costs(a, pre);
        const int64_t total = (int64_t)pre[a.B] * per_b, share = share_of();
        Line x = {};
        x.at = min(total, (int64_t)blockIdx.x * share);
        x.end = min(total, x.at + share);
        if (threadIdx.x == 0) a.chain[2 * blockIdx.x + 1] = 0;
        if (x.at < x.end) {
            int hi = a.B;  // pre[b] * per_b <= at < pre[b + 1] * per_b
            while (hi - x.b > 1) {
                const int mid = (x.b + hi) >> 1;
                if ((int64_t)pre[mid] * per_b <= x.at) x.b = mid;
                else hi = mid;
            }
            const int64_t off = x.at - (int64_t)pre[x.b] * per_b;
            const int cost = pre[x.b + 1] - pre[x.b];
            x.item = (int)(off / cost);
            x.into = (int)(off - (int64_t)x.item * cost);
        }
        if (lane == 0) *line = x;
    } else if (lane == 0) {
        Line x = {};
        x.end = 1;  // the CTA's one item is still to come
        const int i = JOINT ? blockIdx.x / a.cluster : blockIdx.x;
        x.b = i / per_b;
        x.item = i - x.b * per_b;
        *line = x;
    }
    __syncwarp();
    // The next part, by lane 0 into line->next.
    auto step = [&]() {
        if (lane == 0) {
            Line y = *line;
            Part& x = y.next;
            x.n = -1;
            if (JOINT || !a.split) {
                if (y.at < y.end) {
                    const int n = Seen(a, y.b).n;
                    x = {y.b, y.item, 0, n, n};
                    if constexpr (JOINT) {
                        const int r = blockIdx.x % a.cluster;
                        x.i0 = (int)((int64_t)n * r / a.cluster);
                        x.n = (int)((int64_t)n * (r + 1) / a.cluster) - x.i0;
                    }
                    y.at = y.end;
                }
            } else {
                while (y.at < y.end) {
                    const int cost = pre[y.b + 1] - pre[y.b];
                    const int stop = (int)min((int64_t)cost, y.into + (y.end - y.at));  // costs come first, then tiles
                    x = {y.b, y.item, max(0, y.into - ITEM_COST), 0, cost - ITEM_COST};
                    const int n = max(0, stop - ITEM_COST) - x.i0;
                    x.n = n > 0 ? n : -1;
                    y.at += stop - y.into;
                    y.into = 0;
                    if (stop == cost && ++y.item == per_b) {
                        y.item = 0;
                        do ++y.b;
                        while (y.at < y.end && pre[y.b + 1] == pre[y.b]);
                    }
                    if (n > 0) break;
                }
            }
            *line = y;
        }
        __syncwarp();
    };

    // ---- the ring ----
    uint32_t used = 0;  // steps this warp has taken from its ring (stage = used % ST)
    int* ahead = reinterpret_cast<int*>(smem + S::AHEAD) + 64 * warp;
    auto tiles_of_warp = [&](const Part& x) { return x.n > warp ? (x.n - warp + WARPS - 1) / WARPS : 0; };
    // Record numbers of tiles 32 block + lane of this warp; -1: none, or no such page.
    auto records = [&](const Part& x, const Seen& seen, int block) {
        const int k = 32 * block + lane;
        if (k >= tiles_of_warp(x)) return -1;
        const int tile = seen.tile(x.i0 + warp + WARPS * k);
        const int page = tile / a.tpp;
        const int id = __ldg(a.table + (int64_t)x.b * a.tb + page);
        if (id < 0 || id >= a.pages) {
            kv4::report(g_kv4_attention_status, kv4::BAD_INDEX, kv4::AT_PAGE);
            return -1;
        }
        return (id * a.Hk + x.item / a.blocks) * a.tpp + (tile - page * a.tpp);
    };
    // Lane 0: the records of step k (-1: none) into its stage.
    auto issue = [&](int k, const int (&rec)[TS]) {
        const uint32_t stage = (used + (uint32_t)k) % ST;
        uint64_t* bar = &bars[warp * ST + stage];
        uint32_t bytes = 0;
#pragma unroll
        for (int u = 0; u < TS; ++u) bytes += rec[u] < 0 ? 0 : R::BYTES;
        if (bytes == 0) {
            sm100::mbar_arrive(bar);
            return;
        }
        sm100::mbar_arrive_expect_tx(bar, bytes);
#pragma unroll
        for (int u = 0; u < TS; ++u)
            if (rec[u] >= 0)
                sm100::bulk_load(sm100::smem_u32(smem) + (warp * ST + stage) * S::STAGE + u * R::BYTES, a.cache + (int64_t)rec[u] * R::BYTES, R::BYTES, bar);
    };
    // A part's first 64 record numbers, looked up long before they are needed.
    auto look_up = [&](const Part& x) {
        if (x.n <= 0) return;
        const Seen seen(a, x.b);
        ahead[lane] = records(x, seen, 0);
        ahead[32 + lane] = records(x, seen, 1);
        __syncwarp();
    };
    int steps, issued, rec_now, rec_next;  // of the warp: steps in the part, steps whose copies are issued
    uint4 raw[NT][NG][2];  // the lane's elements 64 G + 16 t + 0..15 of heads g (+ 8)
    // Begin a part that has been looked up: its first copies and its queries.
    auto begin = [&](const Part& x) {
        if (x.n < 0) return;
        steps = (tiles_of_warp(x) + TS - 1) / TS;
        rec_now = x.n ? ahead[lane] : -1;
        rec_next = x.n ? ahead[32 + lane] : -1;
        for (issued = 0; issued < min(steps, ST - 1); ++issued) {
            int rec[TS];
#pragma unroll
            for (int u = 0; u < TS; ++u) rec[u] = __shfl_sync(0xffffffffu, rec_now, TS * issued + u);
            if (lane == 0) issue(issued, rec);
        }
        const int kh = x.item / a.blocks, hb = x.item - kh * a.blocks;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int G = 0; G < NG; ++G) {
                const int h = hb * HB + nt * 8 + g;
                raw[nt][G][0] = raw[nt][G][1] = make_uint4(0, 0, 0, 0);
                if (h < a.group && steps) {
                    const T* src = (const T*)a.q + (int64_t)x.b * a.qb + (int64_t)(kh * a.group + h) * a.qh + 64 * G + 16 * t;
                    raw[nt][G][0] = *reinterpret_cast<const uint4*>(src);
                    raw[nt][G][1] = *reinterpret_cast<const uint4*>(src + 8);
                }
            }
    };
    step();
    Part now = line->next;
    look_up(now);
    begin(now);

    if (!JOINT && a.split) {  // requests that see nothing belong to no stretch
        for (int e = blockIdx.x; e < a.B; e += gridDim.x)
            if (pre[e + 1] == pre[e])
                for (int i = threadIdx.x; i < a.Hk * a.group * D; i += THREADS)
                    ((T*)a.o)[(int64_t)e * a.ob + (int64_t)(i / D) * a.oh + i % D] = sf::Dt<T>::from_f(0.f);
    }
    if (blockIdx.x == 0 && warp == 0)
        for (int e = lane; e < a.B; e += 32)
            if (__ldg(a.lens + e) > a.width * a.tpp * 16) kv4::report(g_kv4_attention_status, kv4::BAD_INDEX, kv4::AT_LENGTH);
    __syncthreads();  // `merged` is initialised

    for (uint32_t round = 0; now.n >= 0; ++round) {
        const Seen seen(a, now.b);
        const int64_t now_end = line->at;  // behind this part
        __syncwarp();
        step();
        look_up(line->next);
        uint32_t bad = __ballot_sync(0xffffffffu, steps && rec_now < 0);  // of a block of 32 tiles: nothing was copied

        // ---- q as the B operand ----
        uint32_t qf[NT][8 * NG], qlow[NT];
        float2 fac[NT];  // of the lane's columns, heads 2t and 2t + 1
        {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float amax = 0.f, sum[NG];
#pragma unroll
                for (int G = 0; G < NG; ++G) {
                    const uint32_t w[8] = {raw[nt][G][0].x, raw[nt][G][0].y, raw[nt][G][0].z, raw[nt][G][0].w,
                                           raw[nt][G][1].x, raw[nt][G][1].y, raw[nt][G][1].z, raw[nt][G][1].w};
                    float2 two = sf::f2(0.f);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float2 f = sf::Pair<T>::to_f2(w[i]);
                        amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
                        two = sf::f2_fma(f, sf::f2(1.0f / S_UNIT), two);
                    }
                    sum[G] = two.x + two.y;
#pragma unroll
                    for (int o = 1; o <= 2; o <<= 1) sum[G] += __shfl_xor_sync(0xffffffffu, sum[G], o);
                }
#pragma unroll
                for (int o = 1; o <= 2; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
                // Of sum(q_G), G = 0, 1, the lane's t-th bf16 part: t = 0, 1, 2 make up 24 bits.
                float part[2] = {sum[0] * a.scale_log2, NG == 2 ? sum[NG - 1] * a.scale_log2 : 0.f};
                qlow[nt] = 0;
#pragma unroll
                for (int i = 0; i < 3; ++i) {
                    const uint32_t w = sf::Pair<__nv_bfloat16>::from_f2(make_float2(part[0], part[1]));
                    const float2 back = sf::Pair<__nv_bfloat16>::to_f2(w);
                    if (t == i) qlow[nt] = w;
                    part[0] -= back.x;
                    part[1] -= back.y;
                }
                // amax 2^(137 - ex) in [2^10, 2^11): times 16 it is still an fp16.  The least exponent keeps 16 up
                // finite; an infinity takes the largest and turns its own head into NaN.
                const uint32_t ex = min(max(__float_as_uint(amax) >> 23, 14u), 254u);
                const float up = __uint_as_float((264u - ex) << 23), up16 = up * 16.f;
                const float mine = __uint_as_float(ex << 23) * a.scale_log2;  // 2^(ex - 137) 2^20 / S_UNIT, head g's
                fac[nt] = make_float2(__shfl_sync(0xffffffffu, mine, 8 * t), __shfl_sync(0xffffffffu, mine, 8 * t + 4));
#pragma unroll
                for (int G = 0; G < NG; ++G)
#pragma unroll
                    for (int h2 = 0; h2 < 2; ++h2) {
                        const uint4 r4 = raw[nt][G][h2];
                        const float2 e01 = sf::Pair<T>::to_f2(r4.x), e23 = sf::Pair<T>::to_f2(r4.y), e45 = sf::Pair<T>::to_f2(r4.z),
                                     e67 = sf::Pair<T>::to_f2(r4.w);
                        uint32_t* f = &qf[nt][(2 * G + h2) * 4];
                        f[0] = f16x2(e01.x * up16, e45.x * up16);
                        f[1] = f16x2(e01.y * up, e45.y * up);
                        f[2] = f16x2(e23.x * up16, e67.x * up16);
                        f[3] = f16x2(e23.y * up, e67.y * up);
                    }
            }
        }

        // O^T, heads 2t, 2t + 1, elements 64 G + 8 g + 4 i + 0..3 for i < 2: [4 G + i] whole bytes (rows g
        // and g + 8 are the lower and upper pair of elements), [4 G + 2 + i] their upper codes times 16.
        float o[NT][4 * NG][4];
        float2 nm[NT], l[NT], pm[NT][NG];  // minus the max that weights are relative to, their sum, sum p (minimum + 8 scale)
        float2 unit[NT], per_unit[NT];     // O is in this unit, a head each; the largest p s is at most UNITS_MOST of it
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int i = 0; i < 4 * NG; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c) o[nt][i][c] = 0.f;
            nm[nt] = sf::f2(-NO_MAX);
            l[nt] = sf::f2(0.f);
            unit[nt] = sf::f2(UNIT_FLOOR);
            per_unit[nt] = sf::f2(1.0f / UNIT_FLOOR);
#pragma unroll
            for (int G = 0; G < NG; ++G) pm[nt][G] = sf::f2(0.f);
        }

        // ---- the warp's tiles ----
        const uint8_t* ring = smem + warp * ST * S::STAGE;
        // Tiles that may hold keys past either end of what is seen: the last, the last of the sinks and
        // the first behind them.
        const int edge0 = seen.sink_tiles - 1 - now.i0, edge1 = seen.sink_tiles - now.i0, edge2 = seen.n - 1 - now.i0;
        for (int k = 0; k < steps; ++k) {
            if (k && (TS * k & 31) == 0) {
                rec_now = rec_next;
                bad = __ballot_sync(0xffffffffu, rec_now < 0);
                rec_next = records(now, seen, (TS * k >> 5) + 1);
            }
            __syncwarp();  // every lane is done with the stage that the next copy overwrites
            if (issued < steps) {
                const int from = TS * issued >> 5 == TS * k >> 5 ? rec_now : rec_next;
                int rec[TS];
#pragma unroll
                for (int u = 0; u < TS; ++u) rec[u] = __shfl_sync(0xffffffffu, from, (TS * issued + u) & 31);
                if (lane == 0) issue(issued, rec);
                ++issued;
            }
            const uint32_t turn = used + (uint32_t)k;
            // A copy that never lands leaves its status; the numbers are void then, and the waits that
            // follow end early.
            sm100::mbar_wait(&bars[warp * ST + turn % ST], (turn / ST) & 1u, g_kv4_attention_status + 1, kv4::AT_WAIT);
            __syncwarp();
            const uint32_t none = bad >> (TS * k & 31);
            if ((none & ((1u << TS) - 1u)) == (1u << TS) - 1u) continue;
            const uint8_t* rec = ring + (turn % ST) * S::STAGE;

            // Scales and minima of the lane's keys `row` and `row + 8` of each tile.
            uint32_t vp[TS][2][NG];
            float s[TS][NT][4];  // S^T: [row, row + 8] x heads 2t, 2t + 1
#pragma unroll
            for (int u = 0; u < TS; ++u) {
                const uint8_t* tile = rec + u * R::BYTES;
                uint32_t kp[2][NG], kw[2][2 * NG];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const uint8_t* p = tile + R::K + (row + 8 * r) * R::ROW + t * 8 * NG;
                    if constexpr (NG == 2) {
                        *reinterpret_cast<uint2*>(kp[r]) = *reinterpret_cast<const uint2*>(tile + R::KP + (row + 8 * r) * 8);
                        *reinterpret_cast<uint2*>(vp[u][r]) = *reinterpret_cast<const uint2*>(tile + R::VP + (row + 8 * r) * 8);
                        *reinterpret_cast<uint4*>(kw[r]) = *reinterpret_cast<const uint4*>(p);
                    } else {
                        kp[r][0] = *reinterpret_cast<const uint32_t*>(tile + R::KP + (row + 8 * r) * 4);
                        vp[u][r][0] = *reinterpret_cast<const uint32_t*>(tile + R::VP + (row + 8 * r) * 4);
                        *reinterpret_cast<uint2*>(kw[r]) = *reinterpret_cast<const uint2*>(p);
                    }
                }
                // S^T = K q^T: the minima's part, then a group at a time.
                float2 codes[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    mma_bf16_k8_first(s[u][nt], NG == 2 ? __byte_perm(kp[0][0], kp[0][NG - 1], 0x7632) : kp[0][0] >> 16,
                                      NG == 2 ? __byte_perm(kp[1][0], kp[1][NG - 1], 0x7632) : kp[1][0] >> 16, qlow[nt]);
#pragma unroll
                for (int G = 0; G < NG; ++G) {
                    float acc[NT][4];
#pragma unroll
                    for (int h2 = 0; h2 < 2; ++h2) {
                        const uint32_t x = kw[0][2 * G + h2], y = kw[1][2 * G + h2], x8 = x >> 8, y8 = y >> 8;
                        const uint32_t a0[4] = {x & 0x000F000Fu, y & 0x000F000Fu, x & 0x00F000F0u, y & 0x00F000F0u};
                        const uint32_t a1[4] = {x8 & 0x000F000Fu, y8 & 0x000F000Fu, x8 & 0x00F000F0u, y8 & 0x00F000F0u};
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            const uint32_t* f = &qf[nt][(2 * G + h2) * 4];
                            if (h2 == 0) mma_f16_first(acc[nt], a0, f[0], f[1]);
                            else mma_f16(acc[nt], a0, f[0], f[1]);
                            mma_f16(acc[nt], a1, f[2], f[3]);
                        }
                    }
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const float2 ks = sf::f2(__uint_as_float(kp[r][G] << 16));
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            const float2 x = make_float2(acc[nt][2 * r], acc[nt][2 * r + 1]);
                            codes[nt][r] = G == 0 ? sf::f2_mul(x, ks) : sf::f2_fma(x, ks, codes[nt][r]);
                        }
                    }
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const float2 x = sf::f2_fma(codes[nt][r], fac[nt], make_float2(s[u][nt][2 * r], s[u][nt][2 * r + 1]));
                        s[u][nt][2 * r] = x.x;
                        s[u][nt][2 * r + 1] = x.y;
                    }
                const int at_tile = warp + WARPS * (TS * k + u);
                if (at_tile == edge0 || at_tile == edge1 || at_tile == edge2 || (none >> u & 1u)) {
                    const int j = seen.tile(now.i0 + at_tile) * 16 + row;
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        if (!(none >> u & 1u) && j + 8 * r < seen.len && (j + 8 * r >= seen.low || j + 8 * r < a.sinks)) continue;
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) s[u][nt][2 * r] = s[u][nt][2 * r + 1] = -INFINITY;
#pragma unroll
                        for (int G = 0; G < NG; ++G) vp[u][r][G] = 0;
                    }
                }
            }
            // The running max follows only when a score passes it by 2^8: p stays within fp32 and fp16
            // range and the final division takes the stale max out again.  O follows through its unit.
            float over = -INFINITY;
#pragma unroll
            for (int u = 0; u < TS; ++u)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int r = 0; r < 2; ++r)
                        over = fmaxf(over, fmaxf(fmaf(s[u][nt][2 * r], S_UNIT, nm[nt].x), fmaf(s[u][nt][2 * r + 1], S_UNIT, nm[nt].y)));
            if (__any_sync(0xffffffffu, over > 8.f)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float2 mx = make_float2(fmaxf(s[0][nt][0], s[0][nt][2]), fmaxf(s[0][nt][1], s[0][nt][3]));
                    if constexpr (TS == 2)
                        mx = make_float2(fmaxf(mx.x, fmaxf(s[TS - 1][nt][0], s[TS - 1][nt][2])), fmaxf(mx.y, fmaxf(s[TS - 1][nt][1], s[TS - 1][nt][3])));
                    mx = over_keys(mx);
                    mx = make_float2(fmaxf(mx.x * S_UNIT, -nm[nt].x), fmaxf(mx.y * S_UNIT, -nm[nt].y));
                    const float2 f = make_float2(exp2f(-nm[nt].x - mx.x), exp2f(-nm[nt].y - mx.y));
                    nm[nt] = make_float2(-mx.x, -mx.y);
                    l[nt] = sf::f2_mul(l[nt], f);
                    unit[nt] = sf::f2_mul(unit[nt], f);
                    // A unit that vanishes takes along what it counted.
                    unit[nt] = make_float2(fmaxf(unit[nt].x, UNIT_FLOOR), fmaxf(unit[nt].y, UNIT_FLOOR));
                    per_unit[nt] = make_float2(1.0f / unit[nt].x, 1.0f / unit[nt].y);
#pragma unroll
                    for (int G = 0; G < NG; ++G) pm[nt][G] = sf::f2_mul(pm[nt][G], f);
                }
            }
            // p over the scores, its sum, and the largest p s in O's unit.
            over = 0.f;
#pragma unroll
            for (int u = 0; u < TS; ++u)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    float vs[NG], vm[NG];
#pragma unroll
                    for (int G = 0; G < NG; ++G) {
                        vs[G] = __uint_as_float(vp[u][r][G] << 16);
                        vm[G] = fmaf(8.f, vs[G], __uint_as_float(vp[u][r][G] & 0xFFFF0000u));
                    }
                    const float top = NG == 2 ? fmaxf(vs[0], vs[NG - 1]) : vs[0];
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float2 p = sf::f2_fma(make_float2(s[u][nt][2 * r], s[u][nt][2 * r + 1]), sf::f2(S_UNIT), nm[nt]);
                        p = make_float2(sf::ex2_ftz(p.x), sf::ex2_ftz(p.y));
                        l[nt] = sf::f2_add(l[nt], p);
#pragma unroll
                        for (int G = 0; G < NG; ++G) pm[nt][G] = make_float2(fmaf(p.x, vm[G], pm[nt][G].x), fmaf(p.y, vm[G], pm[nt][G].y));
                        const float2 pu = sf::f2_mul(p, per_unit[nt]);
                        over = fmaxf(over, fmaxf(pu.x * top, pu.y * top));
                        s[u][nt][2 * r] = p.x;
                        s[u][nt][2 * r + 1] = p.y;
                    }
                }
            if (__any_sync(0xffffffffu, over > UNITS_MOST)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float2 top = sf::f2(0.f);  // the head's largest p s
#pragma unroll
                    for (int u = 0; u < TS; ++u)
#pragma unroll
                        for (int r = 0; r < 2; ++r)
#pragma unroll
                            for (int G = 0; G < NG; ++G) {
                                const float vs = __uint_as_float(vp[u][r][G] << 16);
                                top = make_float2(fmaxf(top.x, s[u][nt][2 * r] * vs), fmaxf(top.y, s[u][nt][2 * r + 1] * vs));
                            }
                    top = over_keys(top);
                    // Where this head's own weights fit, its unit stays.
                    const float2 un = make_float2(top.x > UNITS_MOST * unit[nt].x ? fmaxf(top.x * (1.0f / UNITS_NEW), UNIT_FLOOR) : unit[nt].x,
                                                  top.y > UNITS_MOST * unit[nt].y ? fmaxf(top.y * (1.0f / UNITS_NEW), UNIT_FLOOR) : unit[nt].y);
                    per_unit[nt] = make_float2(1.0f / un.x, 1.0f / un.y);
                    const float2 f = sf::f2_mul(unit[nt], per_unit[nt]);
                    unit[nt] = un;
#pragma unroll
                    for (int i = 0; i < 4 * NG; ++i) {
                        o[nt][i][0] *= f.x;
                        o[nt][i][1] *= f.y;
                        o[nt][i][2] *= f.x;
                        o[nt][i][3] *= f.y;
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < TS; ++u) {
                const uint8_t* tile = rec + u * R::BYTES;
                uint32_t pf[NT][NG][PARTS][2];  // p s in O's unit, the B operand of O^T = V^T p^T
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const float2 pu = sf::f2_mul(make_float2(s[u][nt][2 * r], s[u][nt][2 * r + 1]), per_unit[nt]);
#pragma unroll
                        for (int G = 0; G < NG; ++G) {
                            const float vs = __uint_as_float(vp[u][r][G] << 16);
                            const float2 ps = sf::f2_mul(pu, sf::f2(vs));
                            const uint32_t high = f16x2(ps.x, ps.y);
                            pf[nt][G][0][r] = transpose8(high);
                            if constexpr (PARTS == 2) {
                                const float2 rest = sf::f2_fma(sf::Pair<__half>::to_f2(high), sf::f2(-1.f), ps);
                                pf[nt][G][PARTS - 1][r] = transpose8(f16x2(rest.x, rest.y));
                            }
                        }
                    }
                // O^T += V^T p^T: the lane reads its 8 elements a group of keys t, 7 - t, 8 + t, 15 - t.
                uint32_t vw[4][NG];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = (i & 1 ? 7 - t : t) + 8 * (i >> 1);
                    const uint8_t* p = tile + R::V + key * R::ROW + (g ^ (4 * ((key >> 1) & 1))) * 4 * NG;
                    if constexpr (NG == 2) {
                        *reinterpret_cast<uint2*>(vw[i]) = *reinterpret_cast<const uint2*>(p);
                    } else {
                        vw[i][0] = *reinterpret_cast<const uint32_t*>(p);
                    }
                }
#pragma unroll
                for (int G = 0; G < NG; ++G)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        // Elements 4 i .. 4 i + 3 (two bytes) of two keys side by side in the halves of a word.
                        const uint32_t y = __byte_perm(vw[0][G], vw[1][G], i ? 0x7632 : 0x5410), w = __byte_perm(vw[2][G], vw[3][G], i ? 0x7632 : 0x5410);
                        const uint32_t b[4] = {(y & 0x00FF00FFu) | 0x64006400u, __byte_perm(y, 0x64646464u, 0x4341), (w & 0x00FF00FFu) | 0x64006400u,
                                               __byte_perm(w, 0x64646464u, 0x4341)};
                        uint32_t all[4], up[4];
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            all[c] = sub2(b[c], 0x64886488u);                 // 1024 + byte - 1160
                            up[c] = sub2(b[c] & 0xFFF0FFF0u, 0x64806480u);    // 1024 + 16 code - 1152
                        }
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int part = 0; part < PARTS; ++part) {
                                mma_f16(o[nt][4 * G + i], all, pf[nt][G][part][0], pf[nt][G][part][1]);
                                mma_f16(o[nt][4 * G + 2 + i], up, pf[nt][G][part][0], pf[nt][G][part][1]);
                            }
                    }
            }
        }
        used += (uint32_t)steps;

        // ---- the warps' states side by side, then one sum over them ----
        if (round) sm100::mbar_wait(merged, (round - 1) & 1u, g_kv4_attention_status + 1, kv4::AT_WAIT);
        __syncwarp();
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) {
                l[nt].x += __shfl_xor_sync(0xffffffffu, l[nt].x, off);
                l[nt].y += __shfl_xor_sync(0xffffffffu, l[nt].y, off);
#pragma unroll
                for (int G = 0; G < NG; ++G) {
                    pm[nt][G].x += __shfl_xor_sync(0xffffffffu, pm[nt][G].x, off);
                    pm[nt][G].y += __shfl_xor_sync(0xffffffffu, pm[nt][G].y, off);
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int head = nt * 8 + 2 * t + h;
                if (g == 0)
                    *reinterpret_cast<float2*>(stat_s + (warp * HB + head) * 2) = make_float2(h ? -nm[nt].y : -nm[nt].x, h ? l[nt].y : l[nt].x);
                float* dst = out_s + (warp * HB + head) * S::PAD + 8 * g;
#pragma unroll
                for (int G = 0; G < NG; ++G) {
                    const float add = h ? pm[nt][G].y : pm[nt][G].x, u = h ? unit[nt].y : unit[nt].x;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float *all = o[nt][4 * G + i], *up = o[nt][4 * G + 2 + i];
                        *reinterpret_cast<float4*>(dst + 64 * G + 4 * i) =
                            make_float4(fmaf(all[h] - up[h], u, add), fmaf(up[h], u * 0.0625f, add), fmaf(all[h + 2] - up[h + 2], u, add),
                                        fmaf(up[h + 2], u * 0.0625f, add));
                    }
                }
            }
        }
        const Part done = now;
        now = line->next;
        begin(now);
        __syncthreads();
        const bool all_mine = done.n == done.whole;
        const int kh = done.item / a.blocks, hb = done.item - kh * a.blocks;
        const int slot = 2 * blockIdx.x + (done.i0 > 0 ? 0 : 1);
        const int active = min(done.n, WARPS);  // warps that had tiles
        for (int e = threadIdx.x; e < HB * (D / 4); e += THREADS) {
            const int head = e / (D / 4), d = 4 * (e % (D / 4));
            float mx = NO_MAX, sum = 0.f, mw[WARPS];
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                mw[w] = w < active ? stat_s[(w * HB + head) * 2] : NO_MAX;
                mx = fmaxf(mx, mw[w]);
            }
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                if (w >= active) break;
                const float f = exp2f(mw[w] - mx);
                const float4 y = *reinterpret_cast<const float4*>(out_s + (w * HB + head) * S::PAD + d);
                sum = fmaf(f, stat_s[(w * HB + head) * 2 + 1], sum);
                acc.x = fmaf(f, y.x, acc.x);
                acc.y = fmaf(f, y.y, acc.y);
                acc.z = fmaf(f, y.z, acc.z);
                acc.w = fmaf(f, y.w, acc.w);
            }
            if constexpr (JOINT) {
                *reinterpret_cast<float4*>(out_s + head * S::PAD + d) = acc;  // warp 0's place, which no other thread reads
                if (d == 0) *reinterpret_cast<float2*>(smem + S::MERGED + 8 * head) = make_float2(mx, sum);
            } else if (all_mine) {
                if (hb * HB + head < a.group) {
                    const float inv = sum == 0.f ? 0.f : 1.0f / sum;  // 0: every key was hidden
                    T* dst = (T*)a.o + (int64_t)done.b * a.ob + (int64_t)(kh * a.group + hb * HB + head) * a.oh + d;
                    *reinterpret_cast<uint2*>(dst) = make_uint2(sf::Pair<T>::from_f2(make_float2(acc.x * inv, acc.y * inv)),
                                                                sf::Pair<T>::from_f2(make_float2(acc.z * inv, acc.w * inv)));
                }
            } else {
                *reinterpret_cast<float4*>(a.part + ((int64_t)slot * HB + head) * D + d) = acc;
                if (d == 0) *reinterpret_cast<float2*>(a.stat + ((int64_t)slot * HB + head) * 2) = make_float2(mx, sum);
            }
        }
        // An item that starts here and goes on in the CTAs behind is joined from here.
        if (!JOINT && threadIdx.x == 0 && done.i0 == 0 && !all_mine) {
            const int64_t share = share_of();
            a.chain[2 * blockIdx.x] = done.b * per_b + done.item;
            a.chain[2 * blockIdx.x + 1] = (int)((now_end - done.n + done.whole - 1) / share) - blockIdx.x + 1;
        }
        __syncwarp();
        if (lane == 0) sm100::mbar_arrive(merged);
    }

    // ---- a cluster's states, each CTA a share of the elements ----
    if constexpr (JOINT) {
        __syncwarp();
        sm100::cluster_sync();
        const int i = blockIdx.x / a.cluster, b = i / per_b, kh = (i - b * per_b) / a.blocks, hb = i - b * per_b - kh * a.blocks;
        const int rank = blockIdx.x % a.cluster;
        for (int e = rank * THREADS + threadIdx.x; e < HB * D / 2; e += a.cluster * THREADS) {
            const int head = e / (D / 2), d = 2 * (e % (D / 2));
            if (hb * HB + head >= a.group) break;  // heads come in order
            const uint32_t out_at = sm100::smem_u32(out_s + head * S::PAD + d), stat_at = sm100::smem_u32(smem + S::MERGED + 8 * head);
            float mx = NO_MAX, sum = 0.f;
            float2 acc = sf::f2(0.f);
#pragma unroll 4
            for (int r = 0; r < a.cluster; ++r) {
                const float2 st = ld_cluster(sm100::mapa_shared(stat_at, r)), x = ld_cluster(sm100::mapa_shared(out_at, r));
                const float mn = fmaxf(mx, st.x), f = exp2f(mx - mn), g2 = exp2f(st.x - mn);
                mx = mn;
                sum = sum * f + st.y * g2;
                acc = make_float2(acc.x * f + x.x * g2, acc.y * f + x.y * g2);
            }
            const float inv = sum == 0.f ? 0.f : 1.0f / sum;
            *reinterpret_cast<uint32_t*>((T*)a.o + (int64_t)b * a.ob + (int64_t)(kh * a.group + hb * HB + head) * a.oh + d) =
                sf::Pair<T>::from_f2(make_float2(acc.x * inv, acc.y * inv));
        }
        __syncwarp();
        sm100::cluster_sync();  // nobody leaves while its states are read
    }
}

// Join the pieces of the items that span CTAs: blocks of JOIN_HEADS heads of a first CTA's item (spread over
// SMs, since one SM alone takes a microsecond to fetch the pieces), JOIN warps a head, each over every
// JOIN-th piece.
constexpr int JOIN = 4, JOIN_HEADS = 1;
template <typename T, int D, int HB>
__global__ void __launch_bounds__(32 * JOIN_HEADS * JOIN) kv4_join_kernel(const Args a) {
    constexpr int E = D / 32;
    __shared__ float acc_s[JOIN_HEADS][JOIN][D], l_s[JOIN_HEADS][JOIN];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int first = blockIdx.x, hs = threadIdx.x / (32 * JOIN), head = blockIdx.y * JOIN_HEADS + hs, part = (threadIdx.x >> 5) % JOIN, lane = threadIdx.x & 31;
    const int2 chain = *reinterpret_cast<const int2*>(a.chain + 2 * first);
    const int pieces = chain.y, item = chain.x;
    if (pieces == 0) return;
    const int per_b = a.Hk * a.blocks;
    const int b = item / per_b, kh = (item - b * per_b) / a.blocks, hb = item - b * per_b - kh * a.blocks;
    const bool there = hb * HB + head < a.group;
    // The first piece is its CTA's last part, the others their CTAs' first.
    auto slot = [&](int p) { return ((int64_t)2 * (first + p) + (p == 0 ? 1 : 0)) * HB + head; };
    float m = NO_MAX, l = 0.f, acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
    if (there) {
        for (int p = lane; p < pieces; p += 32) m = fmaxf(m, a.stat[slot(p) * 2]);
        m = sf::warp_max(m);
#pragma unroll 4
        for (int p = part; p < pieces; p += JOIN) {
            const float2 st = *reinterpret_cast<const float2*>(a.stat + slot(p) * 2);
            float x[E];
            if constexpr (E == 4) *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(a.part + slot(p) * D + E * lane);
            else *reinterpret_cast<float2*>(x) = *reinterpret_cast<const float2*>(a.part + slot(p) * D + E * lane);
            const float f = exp2f(st.x - m);
            l = fmaf(f, st.y, l);
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] = fmaf(f, x[e], acc[e]);
        }
#pragma unroll
        for (int e = 0; e < E; ++e) acc_s[hs][part][E * lane + e] = acc[e];
        if (lane == 0) l_s[hs][part] = l;
    }
    __syncthreads();
    if (!there || part) return;
#pragma unroll
    for (int w = 1; w < JOIN; ++w) {
        l += l_s[hs][w];
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] += acc_s[hs][w][E * lane + e];
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l;  // 0: every key was hidden
    T* out = (T*)a.o + (int64_t)b * a.ob + (int64_t)(kh * a.group + hb * HB + head) * a.oh + E * lane;
#pragma unroll
    for (int e = 0; e < E; e += 2) *reinterpret_cast<uint32_t*>(out + e) = sf::Pair<T>::from_f2(make_float2(acc[e] * inv, acc[e + 1] * inv));
}

// Most tiles a request can see, from the table's width, window and sinks alone.
int64_t most_tiles(int64_t width, int64_t tpp, int64_t window, int64_t sinks) {
    const int64_t all = width * tpp;
    if (!window || window >= 16 * all || sinks >= 16 * all) return all;
    return std::min(all, (window + 15) / 16 + 1 + (sinks + 15) / 16);
}

// CTAs of the line kernel an SM holds: the prefix of the requests' costs is part of its shared memory, and above some 740
// requests (D 128, one head tile) a third CTA no longer fits into the SM's 228 KB (1 KB a CTA is the system's): 800 requests of up
// to 2048 tokens 445 us with three an SM in the grid, 335 with two.
int64_t resident(int nt, int64_t D, int64_t B) {
    const int b = (int)std::min<int64_t>(B, 1 << 20);
    const int smem = D == 64 ? (nt == 1 ? Smem<1, 1>::bytes(b) : Smem<1, 2>::bytes(b)) : (nt == 1 ? Smem<2, 1>::bytes(b) : Smem<2, 2>::bytes(b));
    return std::max(1, std::min(ctas_of(nt), 228 * 1024 / (smem + 1024)));
}

struct Plan {
    int nt, blocks;
    bool split;
    int cluster, grid;
};

Plan plan_of(int64_t B, int64_t Hq, int64_t Hk, int64_t D, int64_t width, int64_t tpp, int64_t window, int64_t sinks, int32_t variant) {
    Plan p;
    const int64_t group = Hq / Hk;
    p.nt = group > 8 ? 2 : 1;
    p.blocks = (int)((group + 8 * p.nt - 1) / (8 * p.nt));
    const int64_t items = B * Hk * p.blocks;
    const int64_t sms = sf::sm_count(), wave = sms * ctas_of(p.nt);
    const int64_t tiles = most_tiles(width, tpp, window, sinks);
    // Whole items a CTA while an item is at most four tiles a warp: nothing to join.  Longer items of a small
    // batch go to clusters of CTAs that join through each other's shared memory, without a second launch, as
    // long as their stretches are short and the clusters, each of which one group of SMs has to hold, take
    // up to three quarters of the places (16 clusters of 16 on 296 places ran in two rounds: 17.4 against
    // 12.0 us).  Else items are cut so that every CTA gets the same number of tiles.  (Above 1024 requests
    // the items balance the CTAs by themselves, and the prefix of the costs would take the shared memory.)
    p.cluster = 1;
    p.split = tiles > LEAST && B <= 1024;
    if (variant == 0 && p.split) {
        int c = MAX_CLUSTER;
        while (c > 1 && (4 * items * c > 3 * wave || tiles < c * CLUSTER_LEAST)) c /= 2;
        if (c > 1 && tiles <= (int64_t)c * CLUSTER_MOST) p.cluster = c, p.split = false;
    }
    if (variant == 3) p.split = false;
    if (variant == 1) p.split = true;
    p.grid = (int)(p.split ? std::min(sms * resident(p.nt, D, B), std::max<int64_t>(1, (items * (tiles + ITEM_COST) + LEAST - 1) / LEAST)) : items * p.cluster);
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
            cudaError_t e = cudaFuncSetAttribute(kv4_attention_kernel<T, NG, NT, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_SMEM);
            if (e == cudaSuccess) e = cudaFuncSetAttribute(kv4_attention_kernel<T, NG, NT, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_SMEM);
            if (e == cudaSuccess) e = cudaFuncSetAttribute(kv4_attention_kernel<T, NG, NT, true>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
            if (e != cudaSuccess) return sf::fail(SF_EDEVICE, err, cap, "kv4_attention: %s", cudaGetErrorString(e));
            if (dev < 64) done |= 1ull << dev;
        }
    }
    if (p.cluster > 1) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)p.grid);
        cfg.blockDim = dim3(THREADS);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = st;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = p.cluster;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        const cudaError_t e = cudaLaunchKernelEx(&cfg, kv4_attention_kernel<T, NG, NT, true>, (const Args)a);
        if (e != cudaSuccess) return sf::fail(SF_EDEVICE, err, cap, "kv4_attention launch: %s", cudaGetErrorString(e));
        return SF_OK;
    }
    kv4_attention_kernel<T, NG, NT, false><<<p.grid, THREADS, smem, st>>>(a);
    int rc = sf::check_launch("kv4_attention launch", err, cap);
    if (rc || !p.split) return rc;
    // The join starts while the last CTAs of the first kernel run, and waits for all of it.
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)p.grid, (unsigned)((std::min(HB, a.group) + JOIN_HEADS - 1) / JOIN_HEADS));
    cfg.blockDim = dim3(32 * JOIN_HEADS * JOIN);
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
    if (x->variant != 0 && x->variant != 1 && x->variant != 3) return sf::fail(SF_EINVAL, err, cap, "kv4_attention: no variant %d", x->variant);
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
    // The costs of all requests are summed in 32 bits.
    if (B > 0x7fffffffLL / (width * tpp + ITEM_COST)) return sf::fail(SF_EINVAL, err, cap, "kv4_attention: requests x table width too large");
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
    a.cluster = p.cluster;
    const bool half = x->dtype == SF_DTYPE_F16;
    cudaStream_t st = (cudaStream_t)stream;
    if (D == 64) {
        if (p.nt == 1) return half ? launch_t<__half, 1, 1>(a, p, st, err, cap) : launch_t<__nv_bfloat16, 1, 1>(a, p, st, err, cap);
        return half ? launch_t<__half, 1, 2>(a, p, st, err, cap) : launch_t<__nv_bfloat16, 1, 2>(a, p, st, err, cap);
    }
    if (p.nt == 1) return half ? launch_t<__half, 2, 1>(a, p, st, err, cap) : launch_t<__nv_bfloat16, 2, 1>(a, p, st, err, cap);
    return half ? launch_t<__half, 2, 2>(a, p, st, err, cap) : launch_t<__nv_bfloat16, 2, 2>(a, p, st, err, cap);
}
