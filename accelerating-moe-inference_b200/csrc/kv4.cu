// The paged 4-bit key/value cache: block tables and slot maps (plan), the
// quantising append, and attention over the cache.
#include <algorithm>
#include <cmath>
#include <memory>
#include <mutex>
#include <new>
#include <type_traits>
#include <vector>

#include "dtype.cuh"
#include "kv4.cuh"
#include "mma.cuh"
#include "moe_internal.h"

namespace moe {
namespace {

// ------------------------------------------------------------------- plan
// Sums of v over the threads before this one; total the sums over all.  Every
// thread of the block calls it; `buf` holds 33 pairs.
struct Pair {
    long long a, b;
};
__device__ __forceinline__ Pair shfl_up(Pair v, int o) {
    return {__shfl_up_sync(0xffffffffu, v.a, o), __shfl_up_sync(0xffffffffu, v.b, o)};
}
__device__ Pair block_scan(Pair v, Pair* buf, Pair& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    Pair inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const Pair u = shfl_up(inc, o);
        if (lane >= o) inc.a += u.a, inc.b += u.b;
    }
    __syncthreads();
    if (lane == 31) buf[warp] = inc;
    __syncthreads();
    if (warp == 0) {
        const Pair w = lane < warps ? buf[lane] : Pair{0, 0};
        Pair s = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const Pair u = shfl_up(s, o);
            if (lane >= o) s.a += u.a, s.b += u.b;
        }
        buf[lane] = {s.a - w.a, s.b - w.b};
        if (lane == 31) buf[32] = s;
    }
    __syncthreads();
    total = buf[32];
    return {buf[warp].a + inc.a - v.a, buf[warp].b + inc.b - v.b};
}

struct PlanArgs {
    const int* cached;
    const int* added;
    int R, W, bs, nb, cap;
    int* ring;
    const int* state;
    int* table;
    int* kv_len;
    int* q_offset;
    int* position;
    long long* slot;
    int* state_out;
    FastDiv page;     // by bs
};

constexpr int kPlanThreads = 1024;
constexpr int kMaxRequests = 8192;
constexpr size_t plan_smem_bytes(int R) { return (size_t)(2 * R + 1) * sizeof(int); }

// Every block scans all requests (R <= 8192 lengths, L2-resident), so that no
// block waits for another; the requests' rows and the tokens are then split
// over the blocks.  Table entries a token reads lie before the ones written
// here, and pages returned to the ring go behind the ones taken from it, so
// the blocks' reads and writes are disjoint.  Bound by latency: 6.2 us for one
// decode step of 16 requests, 8.2 us for 512 requests and 70 thousand tokens
// (one block for all: 108).
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(PlanArgs a) {
    extern __shared__ int plan_smem[];
    int* q_off = plan_smem;              // [R + 1] clipped to cap
    int* first = plan_smem + a.R + 1;    // [R] first page taken from the ring; -1 rejected; or first page given back
    __shared__ Pair buf[33];
    __shared__ int taken;
    const int per = (a.R + kPlanThreads - 1) / kPlanThreads;
    const int r0 = min(a.R, (int)threadIdx.x * per), r1 = min(a.R, r0 + per);
    int head = a.state[0], count = a.state[1];
    if (head < 0 || head >= a.nb || count < 0 || count > a.nb) head = count = 0;
    const long long limit = (long long)a.W * a.bs;

    if (threadIdx.x == 0) taken = 0;
    // Positions count within pages: 0 <= n <= W * bs <= 2^30.
    auto pages = [&](long long n) { return a.page.div((int)n + a.bs - 1); };
    Pair total, sum{0, 0};
    for (int r = r0; r < r1; ++r) sum.a += max(0, a.added[r]);
    const long long begin = block_scan(sum, buf, total).a, tokens = total.a;
    long long end = begin;
    sum = {0, 0};   // pages needed, pages given back
    for (int r = r0; r < r1; ++r) {
        const long long c = a.cached[r], n = a.added[r];
        q_off[r] = (int)min(end, (long long)a.cap);
        end += max(0ll, n);
        if (c < 0 || c > limit) continue;
        if (n >= 0 && c + n <= limit && (n == 0 || end <= a.cap)) sum.a += pages(c + n) - pages(c);
        if (n < 0) sum.b += pages(c);
    }
    if (threadIdx.x == 0) q_off[a.R] = (int)min(tokens, (long long)a.cap);
    Pair before = block_scan(sum, buf, total);
    const long long given = min(total.b, (long long)a.nb - count);
    end = begin;
    for (int r = r0; r < r1; ++r) {
        const long long c = a.cached[r], n = a.added[r];
        end += max(0ll, n);
        bool ok = false;
        long long take = 0;
        first[r] = -1;
        if (c >= 0 && c <= limit) {
            if (n >= 0 && c + n <= limit && (n == 0 || end <= a.cap)) {
                take = pages(c + n) - pages(c);
                ok = take == 0 || before.a + take <= count;
                if (ok) {
                    first[r] = (int)min(before.a, (long long)count);
                    // The needs of the admitted are a prefix of all needs.
                    if (take) atomicMax(&taken, (int)(before.a + take));
                }
                before.a += take;
            } else if (n < 0) {
                first[r] = (int)min(before.b, given);
                before.b += pages(c);
            }
        }
        if (blockIdx.x == 0) {
            a.kv_len[r] = ok ? (int)(c + n) : 0;
            a.q_offset[r] = q_off[r];
        }
    }
    __syncthreads();
    // Places in the ring are below 2 nb: head < nb, and count plus what is
    // given back is at most nb.
    auto wrap = [&](long long i) { return (int)(i >= a.nb ? i - a.nb : i); };
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        a.q_offset[a.R] = q_off[a.R];
        a.state_out[0] = wrap((long long)head + taken);
        a.state_out[1] = (int)(count - taken + given);
    }

    // The requests' rows: a warp each, 256 pages' loads in flight.
    const int lane = threadIdx.x & 31;
    auto copy = [&](int n, auto from, auto to) {
        for (int i0 = lane; i0 < n; i0 += 256) {
            int v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (i0 + 32 * k < n) v[k] = from(i0 + 32 * k);
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (i0 + 32 * k < n) to(i0 + 32 * k, v[k]);
        }
    };
    const int warps = gridDim.x * (kPlanThreads / 32);
    for (int r = blockIdx.x * (kPlanThreads / 32) + (threadIdx.x >> 5); r < a.R; r += warps) {
        const int f = first[r];
        if (f < 0) continue;
        const long long c = a.cached[r], n = a.added[r];
        const int used = pages(c);
        int* row = a.table + (size_t)r * a.W;
        if (n < 0) {
            copy((int)min((long long)used, given - f), [&](int i) { return row[i]; },
                 [&](int i, int v) { a.ring[wrap((long long)head + count + f + i)] = v; });
        } else {
            const int take = pages(c + n) - used;
            copy(take, [&](int i) { return a.ring[wrap((long long)head + f + i)]; }, [&](int i, int v) { row[used + i] = v; });
        }
    }
    // The tokens: a thread each.  Unsigned: the last step may pass 2^31.
    for (unsigned at = blockIdx.x * kPlanThreads + threadIdx.x; at < (unsigned)a.cap; at += gridDim.x * kPlanThreads) {
        const int t = (int)at;
        int pos = -1;
        long long slot = -1;
        if (t < q_off[a.R]) {
            int lo = 0, hi = a.R - 1;  // the first r with q_off[r + 1] > t
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (q_off[mid + 1] > t) hi = mid;
                else lo = mid + 1;
            }
            const int c = a.cached[lo];
            pos = (int)((unsigned)c + (unsigned)(t - q_off[lo]));   // out of range only where rejected
            if (first[lo] >= 0) {
                const int used = pages(c), b = a.page.div(pos);
                const int page = b < used ? a.table[(size_t)lo * a.W + b]
                                          : a.ring[wrap((long long)head + first[lo] + b - used)];
                if (page >= 0 && page < a.nb) slot = (long long)page * a.bs + pos - b * a.bs;
            }
        }
        a.position[t] = pos;
        a.slot[t] = slot;
    }
}

// ----------------------------------------------------------------- append
// Eight consecutive elements as fp32; kVec: one or two 16-byte loads (the
// address is 16-byte aligned), else element by element.
__device__ __forceinline__ float2 pair_f32(uint32_t v, __nv_bfloat16) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
__device__ __forceinline__ float2 pair_f32(uint32_t v, __half) {
    return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
template <class T, bool kVec> __device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
    if constexpr (kVec && sizeof(T) == 4) {
        const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else if constexpr (kVec) {
        const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = pair_f32(w[i], T{});
            x[2 * i] = f.x, x[2 * i + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_f32(p[i]);
    }
}

// The same as one or two 16-byte stores.
__device__ __forceinline__ uint32_t pair_bits(float a, float b, __nv_bfloat16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pair_bits(float a, float b, __half) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <class T> __device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
    if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
        *reinterpret_cast<uint4*>(p) = make_uint4(pair_bits(x[0], x[1], T{}), pair_bits(x[2], x[3], T{}),
                                                  pair_bits(x[4], x[5], T{}), pair_bits(x[6], x[7], T{}));
    }
}

struct AppendArgs {
    uint8_t* cache;
    const void* x[2];            // k, v
    long long token_stride[2], head_stride[2];
    const long long* slot;
    void* out[2];
    int N, H, bs, nb;
    FastDiv heads;    // by H
    FastDiv page;     // by bs / 16
};

// Range of a group of 64 dims held by 8 neighbouring lanes, 8 dims each; the
// lane's eight codes as a word, their scale and minimum, the values they stand for.
__device__ __forceinline__ uint32_t quantise8(float2 (&x)[4], __half2& param) {
    float lo = fminf(x[0].x, x[0].y), hi = fmaxf(x[0].x, x[0].y);
    float2 sum = x[0];
#pragma unroll
    for (int e = 1; e < 4; ++e) {
        lo = fminf(lo, fminf(x[e].x, x[e].y));
        hi = fmaxf(hi, fmaxf(x[e].x, x[e].y));
        sum = __fadd2_rn(sum, x[e]);
    }
    // A NaN or an infinity shows in the sum, a value out of range in lo or hi.
    unsigned nans = 0;
    const float all = sum.x + sum.y;
    if (__any_sync(0xffffffffu, !(all - all == 0.0f) || lo < -65504.0f || hi > 65504.0f)) {
        bool nan = false;
        lo = 65504.0f, hi = -65504.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            nan |= x[e].x != x[e].x || x[e].y != x[e].y;
            x[e].x = fminf(fmaxf(x[e].x, -65504.0f), 65504.0f);
            x[e].y = fminf(fmaxf(x[e].y, -65504.0f), 65504.0f);
            lo = fminf(lo, fminf(x[e].x, x[e].y));
            hi = fmaxf(hi, fmaxf(x[e].x, x[e].y));
        }
        nans = __ballot_sync(0xffffffffu, nan) >> ((threadIdx.x & 31) & ~7) & 0xff;
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    __half s = __float2half_rn(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f)), z = __float2half_rn(lo);
    if (nans) s = z = __ushort_as_half(0x7fff);
    param = __halves2half2(s, z);
    const float sf = __half2float(s), zf = __half2float(z);
    // The quotient by the approximate reciprocal is off by less than 1e-5; where
    // that could change its rounding the division is done.  Adding 1.5 2^23 rounds
    // to the nearest integer, ties to even, and leaves it in the sum's low bits.
    constexpr float kRound = 12582912.0f;
    const float inv = sf > 0.0f ? rcp_approx(sf) : 0.0f;
    const float2 down = make_float2(-zf, -zf), by = make_float2(inv, inv), round = make_float2(kRound, kRound),
                 back = make_float2(-kRound, -kRound);
    uint32_t word = 0;
    float2 c[4];
    float far = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float2 q = __fmul2_rn(__fadd2_rn(x[e], down), by);
        q.x = fminf(fmaxf(q.x, 0.0f), 15.0f);
        q.y = fminf(fmaxf(q.y, 0.0f), 15.0f);
        const float2 t = __fadd2_rn(q, round);
        c[e] = __fadd2_rn(t, back);
        const float2 off = __ffma2_rn(c[e], make_float2(-1.0f, -1.0f), q);
        far = fmaxf(far, fmaxf(fabsf(off.x), fabsf(off.y)));
        const uint32_t two = __float_as_uint(t.x) & 15u | __float_as_uint(t.y) << 4;   // above 8 bits: kRound's
        word |= (two & 255u) << (8 * e);
    }
    if (far > 0.4999f) {
        word = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            c[e].x = fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(x[e].x, zf), sf)), 0.0f), 15.0f);
            c[e].y = fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(x[e].y, zf), sf)), 0.0f), 15.0f);
            word |= ((uint32_t)c[e].x | (uint32_t)c[e].y << 4) << (8 * e);
        }
    }
    const float2 scale = make_float2(sf, sf), zero = make_float2(zf, zf);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = __ffma2_rn(scale, c[e], zero);   // s * c is exact in fp32
    return word;
}

// A block quantises 16 tokens of one head, a thread 8 dims of K and of V of
// tokens i and i + 8; 8 threads hold a group of 64, so its range is three
// shuffles.  A granule's codes lie in pieces of 4 to 16 bytes per token, so 16
// tokens that fill a granule (a prompt's, from a multiple of 16 on) are put
// together in shared memory and written as whole lines; others (a decode
// step's) are written piece by piece.  A block loads, quantises and stores once,
// so that nothing of its own runs beneath its loads: waiting for them is by far
// the largest stall (4.7 cycles an instruction), 2.5 of 4 instructions are issued
// a cycle, about 25 a value, hence the pairwise fp32 operations.  49 to 50 us for
// 16384 tokens x 8 heads x 128 of bf16 with the values written back, 153 MB at
// 3.1 TB/s (a thread per 8 dims of K or V, with divisions: 86 us).
template <class T, int D, bool kVec> __global__ void __launch_bounds__(D, 1024 / D) append_kernel(AppendArgs a) {
    constexpr int G = D / 64, kThreads = D, kGran = kv4_granule(D);   // D / 8 threads per token
    __shared__ __align__(16) uint8_t stage[kGran];
    const int group = a.heads.div(blockIdx.x), head = blockIdx.x - group * a.H, token0 = group * 16;
    const int m = threadIdx.x % (D / 8), i = threadIdx.x / (D / 8), g = m >> 3;
    float2 x[2][2][4];      // [token][K, V]
    const long long slots = (long long)a.nb * a.bs, slot0 = a.slot[token0];
    long long slot[2];
    bool fits = (slot0 & 15) == 0 && slot0 >= 0 && slot0 < slots;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int token = token0 + i + 8 * h;
        const bool live = token < a.N;
        slot[h] = live ? a.slot[token] : -1;
        fits = fits && slot[h] == slot0 + i + 8 * h;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
            if (live) {
                float v[8];
                load8<T, kVec>(static_cast<const T*>(a.x[kv]) + token * a.token_stride[kv] + head * a.head_stride[kv] + m * 8, v);
#pragma unroll
                for (int e = 0; e < 4; ++e) x[h][kv][e] = make_float2(v[2 * e], v[2 * e + 1]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) x[h][kv][e] = make_float2(0.0f, 0.0f);
            }
        }
    }
    const bool whole = __syncthreads_and(fits);
    auto granule = [&](long long at) {     // of a slot: at / 16 is below 2^31
        const int n = (int)(at >> 4), page = a.page.div(n);
        return a.cache + (((long long)page * a.H + head) * a.page.d + n - page * a.page.d) * kGran;
    };
    // Token i + 8 h's pieces at `gran`, whose offsets from token i's are constants where t is i + 8 h.
    auto put = [&](int h, uint8_t* k_at, uint8_t* v_at, uint8_t* param_at, bool store) {
        const int token = token0 + i + 8 * h;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
            __half2 param;
            const uint32_t word = quantise8(x[h][kv], param);
            if (store) {
                *reinterpret_cast<uint32_t*>(kv == 0 ? k_at : v_at) = word;
                if ((m & 7) == 0) *reinterpret_cast<__half2*>(param_at + kv * 64 * G) = param;
            }
            if (a.out[kv] && token < a.N) {
                const float v[8] = {x[h][kv][0].x, x[h][kv][0].y, x[h][kv][1].x, x[h][kv][1].y,
                                    x[h][kv][2].x, x[h][kv][2].y, x[h][kv][3].x, x[h][kv][3].y};
                store8(static_cast<T*>(a.out[kv]) + ((long long)token * a.H + head) * D + m * 8, v);
            }
        }
    };
    if (whole) {
        uint8_t *k_at = stage + kv4_k_word<D>(i, m), *v_at = stage + kv4_v_word<D>(i, m),
                *param_at = stage + 16 * D + i * G * 4 + g * 4;
        put(0, k_at, v_at, param_at, true);
        put(1, k_at + 4 * D, v_at + (G == 2 ? 512 : 8), param_at + 32 * G, true);   // token i + 8
    } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const bool store = slot[h] >= 0 && slot[h] < slots;
            const int t = (int)(slot[h] & 15);
            uint8_t* gran = store ? granule(slot[h]) : stage;
            put(h, gran + kv4_k_word<D>(t, m), gran + kv4_v_word<D>(t, m), gran + 16 * D + t * G * 4 + g * 4, store);
        }
    }
    if (whole) {
        __syncthreads();
        uint4* to = reinterpret_cast<uint4*>(granule(slot0));
        for (int c = threadIdx.x; c < kGran / 16; c += kThreads) to[c] = reinterpret_cast<const uint4*>(stage)[c];
    }
}

// -------------------------------------------------------------- attention
struct AttendArgs {
    const uint8_t* cache;
    const void* q;
    long long q_token_stride, q_head_stride;
    const int* table;
    const int* kv_len;
    const int* q_offset;
    void* out;
    float* lse;
    float* part;      // [2 * grid][rows of a tile][D + 2]: unnormalised outputs, then m and l
    int* counter;     // [grid], zero between launches
    volatile int* error;   // the handle's, in host memory
    int tokens, H, Hkv, R, W, bs, nb, window;
    float scale;
    bool vec;         // q rows can be read 16 bytes at a time
    FastDiv group;    // by H / Hkv
    FastDiv page;     // by bs / 16
};

constexpr int kAttendWarps = 4;
constexpr int kAttendStages = 3;      // granule pairs in flight per warp
constexpr int kAttendCtasPerSm = 3;
constexpr int kAttendItemCost = 24;   // what an item costs beside its granules, in granules (measured: 25)
constexpr int kAttendMinUnits = 12;   // a block's least share: half a pair of granules a warp more is not worth a join
constexpr int kAttendTop = 14;        // log2 of the largest p s that a row's reference point lets stand
constexpr int kAttendWhole = 8;       // items of up to so many granules are not cut: joining costs more

// What one request asks for: its queries [q0, q0 + nq), cut length, the
// 16-token granules [lo, lo + n) that any of its queries may see, its items
// and their cost.
struct Request {
    int q0, nq, len, lo, n, tiles, items;
    long long units;
};

template <int kRows> __device__ __forceinline__ Request request_of(const AttendArgs& a, int r) {
    Request q;
    q.q0 = min(max(__ldg(a.q_offset + r), 0), a.tokens);
    q.nq = min(max(__ldg(a.q_offset + r + 1), q.q0), a.tokens) - q.q0;
    q.len = (int)min((long long)max(__ldg(a.kv_len + r), 0), (long long)a.W * a.bs);
    q.lo = a.window > 0 ? max(0, q.len - q.nq - a.window + 1) >> 4 : 0;
    q.n = max(1, (int)(((long long)q.len + 15) >> 4) - q.lo);
    const int rows_per_head = q.nq * (a.H / a.Hkv);
    q.tiles = (rows_per_head + kRows - 1) / kRows;
    q.items = a.Hkv * q.tiles;
    q.units = (long long)q.items * (q.n + kAttendItemCost);
    return q;
}

// The code pair at the nibbles `mask` names, as an operand.  As it stands it is
// a pair of subnormals (c 2^-24, or c 2^-20 from the higher nibble of a byte):
// exact, but the tensor core aligns a subnormal's products by its exponent
// field, 2^3 to 2^10 above its value, and drops that much of the sum's low end
// (measured: 5e-6 of the result's norm).  kNormal: made the normal number
// (c - 8) 2^14 times that by one exact fma.  Counted from the middle the terms
// have both signs: a sum of c alone grows to many times the result and is cut
// down to it by the minimums' sum, and what each step of it cut off shows (64
// requests of 100 to 8192 keys: 4e-6 of the result's norm, 1.6e-7 with c - 8).
template <bool kNormal> __device__ __forceinline__ uint32_t codes(uint32_t word, uint32_t mask) {
    uint32_t v = word & mask;
    if constexpr (kNormal) {
        const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&v), __float2half2_rn(16384.0f),
                                  __float2half2_rn(mask == 0x000f000fu ? -8.0f / 1024.0f : -8.0f / 64.0f));
        v = *reinterpret_cast<const uint32_t*>(&r);
    }
    return v;
}

// Where a block stands in its units: the next item is `item` of request r, of
// which `skip` units lie in earlier blocks; `left` units are still the block's.
struct Walk {
    int r, item, skip;
    long long left;
};

// The block's next part of an item: granules [ga, gb) of key/value head `head`
// for one tile of query rows.
struct Segment {
    int r, q0, head, tile, rows;
    int base_pos, pos_lo, pos_hi;    // position of the request's query 0, of the tile's first and last row
    int ga, gb;
    int first, last, n;              // the item's granules that are the block's, of n
    long long before;                // units of the block's before the item's first (may be negative)
};

template <int kRows> __device__ __forceinline__ bool next_segment(const AttendArgs& a, long long share, Walk& w, Segment& g) {
    if (w.left <= 0) return false;
    Request rq = request_of<kRows>(a, w.r);
    while (w.item == rq.items) {         // units are left, so there is a next request
        rq = request_of<kRows>(a, ++w.r);
        w.item = 0;
    }
    const int length = rq.n + kAttendItemCost;
    const long long count = rq.n <= kAttendWhole ? length : min((long long)(length - w.skip), w.left);
    g.first = max(0, w.skip - kAttendItemCost);
    g.last = (int)max(0ll, w.skip + count - kAttendItemCost);
    g.n = rq.n;
    g.before = share - w.left - w.skip;
    const int Gh = a.group.d;
    g.r = w.r;
    g.q0 = rq.q0;
    g.head = rq.tiles == 1 ? w.item : w.item / rq.tiles;
    g.tile = w.item - g.head * rq.tiles;
    g.rows = min(kRows, rq.nq * Gh - g.tile * kRows);
    g.base_pos = rq.len - rq.nq;
    g.pos_lo = g.base_pos + a.group.div(g.tile * kRows);
    g.pos_hi = g.base_pos + a.group.div(g.tile * kRows + g.rows - 1);
    g.ga = rq.lo + g.first;
    g.gb = min(rq.lo + g.last, (g.pos_hi >> 4) + 1);       // pos_hi < 0: none
    if (a.window > 0) g.ga = max(g.ga, max(0, g.pos_lo - a.window + 1) >> 4);
    ++w.item;
    w.skip = 0;
    w.left -= count;
    return g.last > 0;                   // else its granules all lie in later blocks, and the block is done
}

__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Attention over the cache, one pass, the work split evenly over the blocks.
//
// Work: an item is (request, key/value head, tile of query rows); its units are
// kAttendItemCost for what every item costs, then its 16-token granules.  Block
// b takes the units [b * chunk, (b + 1) * chunk) of all items in order, so
// ragged lengths cost no idle blocks and no length is read by the host.  Short
// items stay whole, with the block that has their first unit.  An item that
// lies in several blocks leaves partial (max, sum, output) rows; the block that
// finishes last merges them in order of their place, so the result does not
// depend on the order of arrival.
//
// A warp takes every fourth pair of granules of its block's items and keeps up
// to three pairs in flight by bulk copies into its own ring.  The copies run
// through the block's items without regard to where one ends, so the next
// item's granules are on their way while this one's rows are joined.
//
// Products: m16n8k16 with the cache as A (16 tokens, then 16 dims of the
// transposed values) and the query rows as the 8 columns of B, so that few
// rows (a decode step's heads of one group) fill the product; the
// probabilities of 16 tokens x 8 rows become the second product's B by an 8x8
// transposition between the lanes.  A 4-bit code in the low bits of a float16
// word is the subnormal c 2^-24 (or c 2^-20 four bits higher), so a code pair
// becomes an operand by one AND, exactly (a normal number by one fma more, see
// codes()).  The scale and minimum of a key stand outside
// its product,
//   q . k = s (q . c) + m sum(q),
// those of a value go into the probabilities before the second product,
//   sum_t p_t v_t = sum_t (p_t s_t) c_t + sum_t p_t m_t.
// fp32: with c - 8 in the place of c and m + 8 s in that of m (see codes()).
// Scores are fp32 whatever the type, and lse shows them: of a code at c 2^-24 the
// tensor core cuts off so much that the lse of one key was off by 1.1e-6 for
// float16 queries, six times as far as plain fp32; keys' even nibbles are moved up
// to c 2^-20 first (2.1e-7, attend_long 112 -> 118 us; normal numbers c - 8 for
// every type did the same and cost 2 % more where a request has 8 rows).
// Two planes: fp32 queries, and any type's p s, enter as two float16 numbers, hi
// and (x - hi) 2^11, in neighbouring columns of the same product (22 bits).
// 16-bit types take them where up to four rows leave the columns free, which
// halves the softmax's work too (a lane has one row instead of two: attend_long
// 118 us with one plane, 113 with two).  With one plane p s has 11 bits, and so
// that its rounding counts on c - 7.5 only, not on c, a product with ones gives
// the rounded numbers' sum for float16 results: sum (p s)~ c - 7.5 sum (p s)~ +
// sum p (m + 7.5 s) (8 rows and 100 to 2048 keys: 1.13 times what their own
// rounding leaves instead of 1.75, for 3 % of the time; bfloat16 results, 1.01
// times without it, go without).
//
// Bound by the serial chain of a pair of granules (products, maximum,
// exponentials, products) on the 12 warps an SM that registers and the rings
// leave: about 310 instructions a granule of 2304 bytes, 2.0 of 4 issued a cycle
// with 2.8 warps a scheduler, most stalls on the instruction before.  8 requests
// of 16 k to 131 k tokens, 32 query and 8 key/value heads of 128, f16: 118 us (120
// in a long run), 509 MB at 4.3 TB/s (the copies alone: 85 us); 64 requests of
// 100 to 8192, bf16: 47 us; one of 640, 16 heads, fp32: 12 us.
// NT: column tiles of 8; two take 16 query rows (fp32: 8) per unpacking.
template <class T, int D, int NT, int kPlanes>
__global__ void __launch_bounds__(kAttendWarps * 32, NT == 1 ? kAttendCtasPerSm : 2) attend_kernel(AttendArgs a) {
    constexpr int kRows = 8 * NT / kPlanes;    // query rows of a tile
    constexpr int kE = 2 / kPlanes;            // rows per lane and column tile
    constexpr int kR = kE * NT;                // rows per lane
    constexpr int G = D / 64;
    constexpr int kGran = kv4_granule(D);
    constexpr int kPitch = D + 4;              // floats per output row in shared memory
    constexpr int kThreads = kAttendWarps * 32;
    constexpr float kLo = 1.0f / 2048.0f;      // weight of the low plane
    constexpr bool kNormal = sizeof(T) == 4;   // fp32 results need the whole of their sums
    constexpr bool kOnesSum = kPlanes == 1 && std::is_same_v<T, __half>;   // bf16 results do not show it
    constexpr float kUnit = kNormal ? 64.0f : 1048576.0f;   // what a code of an odd nibble is short of
    constexpr float kCentre = kNormal ? 8.0f : kOnesSum ? 7.5f : 0.0f;   // the code that values are counted from
    constexpr uint32_t kEven = 0x000f000fu, kOdd = 0x00f000f0u;
    constexpr int kStage = 2 * kGran;
    constexpr int kWarpFloats = kRows * kPitch + 2 * kRows;   // a warp's result
    extern __shared__ __align__(16) uint8_t attend_smem[];
    __shared__ Pair scan_buf[33];
    __shared__ long long start_unit;
    __shared__ int start_r, is_last, join_from, join_to;
    __shared__ Walk ahead_walk[kAttendWarps];
    __shared__ uint64_t copies_done[kAttendWarps][kAttendStages];
    __shared__ int2 ahead_run[kAttendWarps], ahead_where[kAttendWarps];

    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, j = lane & 3;
    const int Gh = a.H / a.Hkv;
    uint8_t* ring = attend_smem + warp * kAttendStages * kStage;
    float* results = reinterpret_cast<float*>(attend_smem + kAttendWarps * kAttendStages * kStage);

    // The block's share of the units, and the request its first one lies in.
    const int per = (a.R + kThreads - 1) / kThreads;
    const int r0 = min(a.R, (int)threadIdx.x * per), r1 = min(a.R, r0 + per);
    long long mine = 0;
    for (int r = r0; r < r1; ++r) mine += request_of<kRows>(a, r).units;
    Pair sums;
    long long base = block_scan({mine, 0}, scan_buf, sums).a;
    const long long total = sums.a;
    const long long chunk = max((total + gridDim.x - 1) / gridDim.x, (long long)kAttendMinUnits);
    const long long u0 = blockIdx.x * chunk;
    if (u0 >= total) return;
    if (u0 >= base && u0 < base + mine) {
        for (int r = r0; r < r1; ++r) {
            const long long n = request_of<kRows>(a, r).units;
            if (u0 < base + n) {
                start_r = r;
                start_unit = u0 - base;
                break;
            }
            base += n;
        }
    }
    __syncthreads();
    Walk walk{start_r, 0, 0, min(total - u0, chunk)};
    {
        const Request rq = request_of<kRows>(a, start_r);
        walk.item = (int)(start_unit / (rq.n + kAttendItemCost));
        walk.skip = (int)(start_unit % (rq.n + kAttendItemCost));
        if (walk.skip > 0 && rq.n <= kAttendWhole) {   // the block with its first unit has all of it
            walk.left -= rq.n + kAttendItemCost - walk.skip;
            ++walk.item;
            walk.skip = 0;
        }
    }
    const long long share = min(total - u0, chunk);
    const int page_grans = a.bs >> 4;                          // granules of a head in a page

    // Where the warp's granules lie, up to 16 pairs of one item at a time:
    // lane i holds the place in the cache of the i-th one, kNone without one
    // or where its page is outside the pool; `later` the batch after, loaded
    // ahead.
    constexpr unsigned kNone = 0xffffffffu;
    Walk& ahead = ahead_walk[warp];
    int2& run = ahead_run[warp];          // the granules of the item that are still to be placed
    int2& where = ahead_where[warp];      // its request and head
    if (lane == 0) {
        ahead = walk;
        run = make_int2(0, 0);
    }
    __syncwarp();
    auto locate = [&](int& pairs) {
        int2 left = run, rh = where;
        while (left.x >= left.y) {
            Walk w = ahead;
            Segment sg;
            if (!next_segment<kRows>(a, share, w, sg)) {
                pairs = 0;
                return kNone;
            }
            left = make_int2(sg.ga + 2 * warp, sg.gb);
            rh = make_int2(sg.r, sg.head);
            __syncwarp();
            if (lane == 0) {
                ahead = w;
                where = rh;
            }
            __syncwarp();
        }
        unsigned at = kNone;
        const int gi = left.x + (lane >> 1) * (2 * kAttendWarps) + (lane & 1);
        if (gi < left.y) {
            const int col = a.page.div(gi), page = __ldg(a.table + (size_t)rh.x * a.W + col);
            if (page >= 0 && page < a.nb)
                at = ((unsigned)page * a.Hkv + rh.y) * page_grans + (unsigned)(gi - col * page_grans);
        }
        pairs = min(16, (left.y - left.x + 2 * kAttendWarps - 1) / (2 * kAttendWarps));
        __syncwarp();
        if (lane == 0) run = make_int2(left.x + 32 * kAttendWarps, left.y);
        __syncwarp();
        return at;
    };
    int here_pairs, later_pairs, pair = 0;
    unsigned here = locate(here_pairs), later = locate(later_pairs);
    unsigned valid = 0;    // two bits per stage: there is such a granule
    uint64_t* full = copies_done[warp];   // per stage: its copies have arrived
    unsigned phases = 0;                  // the parity each stage's next wait is for
    bool dead = false;                    // a wait ran out: no more copies
    if (lane == 0) {
#pragma unroll
        for (int i = 0; i < kAttendStages; ++i) mbar_init(full + i, 1);
        fence_mbar_init();
    }
    __syncwarp();
    auto issue = [&](int stage) {
        if (pair == here_pairs) {
            pair = 0;
            here = later;
            here_pairs = later_pairs;
            if (here_pairs) later = locate(later_pairs);
        }
        valid &= ~(3u << (2 * stage));
        if (here_pairs && !dead) {
            const unsigned at0 = __shfl_sync(0xffffffffu, here, 2 * pair), at1 = __shfl_sync(0xffffffffu, here, 2 * pair + 1);
            const unsigned have = (at0 != kNone ? 1u : 0u) | (at1 != kNone ? 2u : 0u);
            valid |= have << (2 * stage);
            if (have && lane == 0) {
                uint8_t* dst = ring + stage * kStage;
                mbar_arrive_expect_tx(full + stage, have == 3 ? kStage : kGran);
                if (have & 1) bulk_load(dst, a.cache + (unsigned long long)at0 * kGran, kGran, full + stage);
                if (have & 2) bulk_load(dst + kGran, a.cache + (unsigned long long)at1 * kGran, kGran, full + stage);
            }
            ++pair;
        }
    };
#pragma unroll
    for (int s = 0; s < kAttendStages - 1; ++s) issue(s);

    int stage = 0;
    Segment sg;
    while (next_segment<kRows>(a, share, walk, sg)) {
        const int rows = sg.rows, tile = sg.tile, head = sg.head;
        // The query fragments: rows scaled by a power of two to below 2^11, for
        // fp32 the dims of even nibbles another 16 up, as their codes are 16 down.
        uint32_t qb[NT][D / 16][2];
        float qs[kR][G], rowf[kR];
        int row_pos[kR];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int local = (n * 8 + g) / kPlanes, row = tile * kRows + local;
            const bool on = local < rows;
            float x[2 * G][8];
            float mx = 0.0f;
            const int tok = a.group.div(row);
            const T* qp = static_cast<const T*>(a.q) + (on ? (sg.q0 + tok) * a.q_token_stride +
                                                              (head * Gh + row - tok * Gh) * a.q_head_stride : 0);
#pragma unroll
            for (int w = 0; w < 2 * G; ++w) {
                const T* p = qp + 64 * (w >> 1) + 16 * j + 8 * (w & 1);
                if (on && a.vec) {
                    load8<T, true>(p, x[w]);
                } else if (on) {
                    load8<T, false>(p, x[w]);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[w][e] = 0.0f;
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(x[w][e]));
            }
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            // Exponent of the largest, kept where 2^(10 - e) is a normal number.
            const int e = min(max((int)(__float_as_uint(mx) >> 23), 11), 253);
            const float up = copysignf(__uint_as_float((264 - e) << 23), a.scale);   // +-2^(10 - (e - 127))
            const float f = fmaxf(fabsf(a.scale) * 1.4426950408889634f * __uint_as_float((e - 10) << 23) * kUnit, 1e-37f);
            float sum[G];
#pragma unroll
            for (int q = 0; q < G; ++q) {
                sum[q] = 0.0f;
#pragma unroll
                for (int w = 2 * q; w < 2 * q + 2; ++w)
#pragma unroll
                    for (int k = 0; k < 8; ++k) sum[q] += x[w][k] *= up;
                sum[q] += __shfl_xor_sync(0xffffffffu, sum[q], 1);
                sum[q] += __shfl_xor_sync(0xffffffffu, sum[q], 2);
                sum[q] *= 1.0f / kUnit;
            }
#pragma unroll
            for (int w = 0; w < 2 * G; ++w)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float k16 = k & 1 || !kNormal ? 1.0f : 16.0f;
                    const float p0 = x[w][k] * k16, p1 = x[w][k + 4] * k16;
                    uint32_t v = half2_bits(p0, p1);
                    if constexpr (kPlanes == 2) {
                        const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&v));
                        if (g & 1) v = half2_bits((p0 - b.x) * 2048.0f, (p1 - b.y) * 2048.0f);
                    }
                    qb[n][2 * w + (k >> 1)][k & 1] = v;
                }
            // What a row's scores need, to the lanes that hold them.
#pragma unroll
            for (int i = 0; i < kE; ++i) {
                const int src = 8 * j + 4 * i;   // lane of column 2 j + i (fp32: 2 j)
                rowf[n * kE + i] = __shfl_sync(0xffffffffu, f, src);
#pragma unroll
                for (int q = 0; q < G; ++q) qs[n * kE + i][q] = __shfl_sync(0xffffffffu, sum[q], src);
                row_pos[n * kE + i] = sg.base_pos + a.group.div(tile * kRows + (n * 8 + 2 * j) / kPlanes + i);
            }
        }

        // Transposed outputs: lane's rows, dims 64 q + 8 g + 2 i (c0, c1) and + 1 (c2, c3).
        float o[NT][G][4][4], all[NT][G][4], m[kR], l[kR], w0[kR][G], off[kR];
#pragma unroll
        for (int i = 0; i < kR; ++i) {
            m[i] = -INFINITY;
            l[i] = off[i] = 0.0f;
#pragma unroll
            for (int q = 0; q < G; ++q) w0[i][q] = 0.0f;
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int q = 0; q < G; ++q)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    all[n][q][c] = 0.0f;
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[n][q][i][c] = 0.0f;
                }

        for (int gi = sg.ga + 2 * warp; gi < sg.gb; gi += 2 * kAttendWarps) {
            const uint8_t* st0 = ring + stage * kStage;
            const unsigned have = valid >> (2 * stage) & 3;
            if (have) {
                if (__any_sync(0xffffffffu, !mbar_wait(full + stage, phases >> stage & 1, nullptr, 0))) {
                    // No more copies; this one gets its time once more, so that
                    // it does not land in memory that is another block's.
                    dead = true;
                    mbar_wait(full + stage, phases >> stage & 1, nullptr, 0);
                    __syncwarp();
                    if (lane == 0) *a.error = kDevErrTimeoutProducer;
                }
                phases ^= 1u << stage;
                // Scores x[row][2 k + h] of the lane's rows and tokens 16 k + g + 8 h.
                float x[kR][4];
                float acc[2][NT][G][4];
                uint32_t kw[2][2][2 * G];   // [granule][half][word]
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint8_t* at = st0 + k * kGran + h * 8 * (D / 2) + lane * (D / 8);
                        if constexpr (G == 2) {
                            const uint4 v = *reinterpret_cast<const uint4*>(at);
                            kw[k][h][0] = v.x, kw[k][h][1] = v.y, kw[k][h][2] = v.z, kw[k][h][3] = v.w;
                        } else {
                            const uint2 v = *reinterpret_cast<const uint2*>(at);
                            kw[k][h][0] = v.x, kw[k][h][1] = v.y;
                        }
                    }
                // The sums of the two granules and groups in turn, so that a
                // product does not wait for the one before it.
#pragma unroll
                for (int step = 0; step < 4; ++step)
#pragma unroll
                    for (int q = 0; q < G; ++q)
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const int w = 2 * q + (step >> 1), shift = 8 * (step & 1);
                            uint32_t f[4];      // 16-bit types: even nibbles moved up to where odd ones are
                            if constexpr (kNormal) {
                                const uint32_t lo = kw[k][0][w] >> shift, hi = kw[k][1][w] >> shift;
                                f[0] = codes<true>(lo, kEven), f[1] = codes<true>(hi, kEven);
                                f[2] = codes<true>(lo, kOdd), f[3] = codes<true>(hi, kOdd);
                            } else {
                                const uint32_t lo = kw[k][0][w], hi = kw[k][1][w];
                                f[0] = (shift ? lo >> 4 : lo << 4) & kOdd, f[1] = (shift ? hi >> 4 : hi << 4) & kOdd;
                                f[2] = lo >> shift & kOdd, f[3] = hi >> shift & kOdd;
                            }
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                const uint32_t(&b)[2] = qb[n][2 * w + (step & 1)];
                                if (step == 0) mma_f16_first(acc[k][n][q], f, b[0], b[1]);
                                else mma_f16(acc[k][n][q], f, b[0], b[1]);
                            }
                        }
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t kp[G];
                        const uint8_t* at = st0 + k * kGran + 16 * D + (g + 8 * h) * G * 4;
                        if constexpr (G == 2) {
                            const uint2 v = *reinterpret_cast<const uint2*>(at);
                            kp[0] = v.x, kp[1] = v.y;
                        } else {
                            kp[0] = *reinterpret_cast<const uint32_t*>(at);
                        }
#pragma unroll
                        for (int i = 0; i < kR; ++i) {
                            float s = 0.0f;
#pragma unroll
                            for (int q = 0; q < G; ++q) {
                                const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&kp[q]));
                                const float (&t)[4] = acc[k][i / kE][q];
                                const float d = kPlanes == 2 ? fmaf(t[2 * h + 1], kLo, t[2 * h]) : t[2 * h + i % kE];
                                const float zero = kNormal ? fmaf(p.x, 8.0f, p.y) : p.y;
                                s = q == 0 ? zero * qs[i][q] : fmaf(zero, qs[i][q], s);
                                s = fmaf(p.x, d, s);
                            }
                            x[i][2 * k + h] = s;
                        }
                    }
                // Value params of the lane's tokens 16 (c / 2) + 8 (c % 2) + g.
                uint32_t vp[4][G];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const uint8_t* at = st0 + (c >> 1) * kGran + 16 * D + 64 * G + (g + 8 * (c & 1)) * G * 4;
                    if constexpr (G == 2) {
                        const uint2 v = *reinterpret_cast<const uint2*>(at);
                        vp[c][0] = v.x, vp[c][1] = v.y;
                    } else {
                        vp[c][0] = *reinterpret_cast<const uint32_t*>(at);
                    }
                }
                const int t0 = gi << 4;
                const bool edge = have != 3 || t0 + 31 > sg.pos_lo || (a.window > 0 && t0 <= sg.pos_hi - a.window);
                unsigned hide = 0;
                if (edge) {
#pragma unroll
                    for (int i = 0; i < kR; ++i)
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const int t = t0 + 8 * c + g;
                            if (!(have >> (c >> 1) & 1) || t > row_pos[i] || (a.window > 0 && t <= row_pos[i] - a.window)) {
                                x[i][c] = -INFINITY;
                                hide |= 1u << (4 * i + c);
                            }
                        }
                }
                // Scores are in units of 1 / rowf, rowf > 0.  The reference point m of
                // a row's exponentials follows score + e, 2^e the power of two at
                // or below the value's scale, so that the second product's operands
                // p s, not p alone, fill float16's range: m moves only when one may
                // lie above 2^14, and then so that the largest is s times a power of
                // two, 2^12 to 2^13: it alone is rounded by next to nothing.
                // Below 2^-14, about 2^-26 of the largest, they lose digits.
                // Scales below 2^-14 count as 2^-15 (p stays below 2^30), a NaN or
                // an infinity too.  Each lane asks by its own tokens' largest e.
                __half2 big = __habs2(*reinterpret_cast<const __half2*>(&vp[0][0]));
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int q = 0; q < G; ++q) big = __hmax2(big, __habs2(*reinterpret_cast<const __half2*>(&vp[c][q])));
                const float lift = (float)((int)(*reinterpret_cast<const uint32_t*>(&big) >> 10 & 31) - (15 + kAttendTop));
                bool above = false;
#pragma unroll
                for (int i = 0; i < kR; ++i)
                    above |= fmaf(fmaxf(fmaxf(x[i][0], x[i][1]), fmaxf(x[i][2], x[i][3])), rowf[i], lift) > m[i];
                if (__any_sync(0xffffffffu, above)) {
                    float e[4];
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        int field = 0;
#pragma unroll
                        for (int q = 0; q < G; ++q) {
                            const int f = vp[c][q] >> 10 & 31;
                            field = max(field, f == 31 ? 0 : f);
                        }
                        e[c] = (float)(field - (15 + kAttendTop));
                    }
#pragma unroll
                    for (int i = 0; i < kR; ++i) {
                        float top = -INFINITY;
#pragma unroll
                        for (int c = 0; c < 4; ++c) top = fmaxf(top, fmaf(x[i][c], rowf[i], e[c]));
#pragma unroll
                        for (int k = 4; k < 32; k <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
                        if (!(top > m[i])) continue;     // the same in the row's lanes
                        const float to = top + 2.0f, keep = exp2_approx(m[i] - to);
                        m[i] = off[i] = to;
                        l[i] *= keep;
#pragma unroll
                        for (int q = 0; q < G; ++q) {
                            w0[i][q] *= keep;
                            if constexpr (kOnesSum) {
                                all[i / kE][q][i % kE] *= keep;
                                all[i / kE][q][2 + i % kE] *= keep;
                            }
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                float (&t)[4] = o[i / kE][q][k];
                                t[i % kE] *= keep;
                                t[2 + i % kE] *= keep;
                                if constexpr (kPlanes == 2) {
                                    t[1] *= keep;
                                    t[3] *= keep;
                                }
                            }
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < kR; ++i) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) x[i][c] = exp2_approx(fmaf(x[i][c], rowf[i], -off[i]));
                    l[i] += (x[i][0] + x[i][1]) + (x[i][2] + x[i][3]);
                }
                // The second product's B: row g, tokens 16 k + 8 h + 2 j, + 1.
                uint32_t pb[2][NT][G][2];
                auto weigh = [&](auto at_edge) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
#pragma unroll
                        for (int q = 0; q < G; ++q) {
                            float2 p = __half22float2(*reinterpret_cast<const __half2*>(&vp[c][q]));
                            if constexpr (kCentre != 0.0f) p.y = fmaf(p.x, kCentre, p.y);
                            float v[kR];
#pragma unroll
                            for (int i = 0; i < kR; ++i) {
                                v[i] = x[i][c] * p.x;
                                if constexpr (at_edge) {   // a hidden token's params may be anything
                                    const bool hidden = hide >> (4 * i + c) & 1;
                                    v[i] = hidden ? 0.0f : v[i];
                                    w0[i][q] += hidden ? 0.0f : x[i][c] * p.y;
                                } else {
                                    w0[i][q] = fmaf(x[i][c], p.y, w0[i][q]);
                                }
                            }
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                uint32_t b;
                                if constexpr (kPlanes == 2) {
                                    const float hi = __half2float(__float2half_rn(v[n]));
                                    b = half2_bits(hi, (v[n] - hi) * 2048.0f);
                                } else {
                                    b = half2_bits(v[2 * n], v[2 * n + 1]);
                                }
                                pb[c >> 1][n][q][c & 1] = transpose8x8(b);
                            }
                        }
                    }
                };
                if (edge) weigh(std::true_type{});
                else weigh(std::false_type{});
                // Values: lane's tokens 2 j, 2 j + 1 of each half, dims 64 q + 8 g + nibble.
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint8_t* st = st0 + k * kGran + 8 * D + lane * 16;
                    uint32_t vw[2][2][G];   // [half][token][group]
                    if constexpr (G == 2) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const uint4 v = *reinterpret_cast<const uint4*>(st + h * 512);
                            vw[h][0][0] = v.x, vw[h][0][1] = v.y, vw[h][1][0] = v.z, vw[h][1][1] = v.w;
                        }
                    } else {
                        const uint4 v = *reinterpret_cast<const uint4*>(st);
                        vw[0][0][0] = v.x, vw[0][1][0] = v.y, vw[1][0][0] = v.z, vw[1][1][0] = v.w;
                    }
#pragma unroll
                    for (int q = 0; q < G; ++q) {
                        if constexpr (kOnesSum) {
                            constexpr uint32_t kOnes[4] = {0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u};
#pragma unroll
                            for (int n = 0; n < NT; ++n) mma_f16(all[n][q], kOnes, pb[k][n][q][0], pb[k][n][q][1]);
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i) {   // byte i: nibbles 2 i (rows g) and 2 i + 1 (rows g + 8)
                            const uint32_t sel = 0x0400 + 0x0101 * i;
                            const uint32_t b0 = __byte_perm(vw[0][0][q], vw[0][1][q], sel);
                            const uint32_t b1 = __byte_perm(vw[1][0][q], vw[1][1][q], sel);
                            const uint32_t f[4] = {codes<kNormal>(b0, kEven), codes<kNormal>(b0, kOdd),
                                                   codes<kNormal>(b1, kEven), codes<kNormal>(b1, kOdd)};
#pragma unroll
                            for (int n = 0; n < NT; ++n) mma_f16(o[n][q][i], f, pb[k][n][q][0], pb[k][n][q][1]);
                        }
                    }
                }
            }
            __syncwarp();
            issue((stage + kAttendStages - 1) % kAttendStages);
            stage = (stage + 1) % kAttendStages;
        }
        // The warp's rows: output, then m and l.
        __syncthreads();   // the last item's are read
        float* res = results + warp * kWarpFloats;
#pragma unroll
        for (int i = 0; i < kR; ++i) {
            const int row = (i / kE * 8 + 2 * j) / kPlanes + i % kE;
#pragma unroll
            for (int k = 4; k < 32; k <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], k);
#pragma unroll
            for (int q = 0; q < G; ++q) {
                float z = w0[i][q];
#pragma unroll
                for (int k = 4; k < 32; k <<= 1) z += __shfl_xor_sync(0xffffffffu, z, k);
                if constexpr (kOnesSum) z = fmaf(all[i / kE][q][i % kE], -kCentre, z);
                float v[8];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float (&t)[4] = o[i / kE][q][k];
                    const float d0 = kPlanes == 2 ? fmaf(t[1], kLo, t[0]) : t[i % kE];
                    const float d1 = kPlanes == 2 ? fmaf(t[3], kLo, t[2]) : t[2 + i % kE];
                    v[2 * k] = fmaf(d0, 16.0f * kUnit, z);
                    v[2 * k + 1] = fmaf(d1, kUnit, z);
                }
                float* to = res + row * kPitch + 64 * q + 8 * g;
                *reinterpret_cast<float4*>(to) = make_float4(v[0], v[1], v[2], v[3]);
                *reinterpret_cast<float4*>(to + 4) = make_float4(v[4], v[5], v[6], v[7]);
            }
            if (g == 0) {
                res[kRows * kPitch + 2 * row] = m[i] == -INFINITY ? -INFINITY : off[i];
                res[kRows * kPitch + 2 * row + 1] = l[i];
            }
        }
        __syncthreads();

        const bool whole = sg.first == 0 && sg.last == sg.n;
        float* part = a.part + (2 * (long long)blockIdx.x + (sg.first == 0 ? 1 : 0)) * kRows * (D + 2);
        auto write = [&](int row, int d, float4 v, float mm, float ll) {
            const int rr = tile * kRows + row;
            const int tok = a.group.div(rr);
            const long long at = (long long)(sg.q0 + tok) * a.H + head * Gh + rr - tok * Gh;
            const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;    // no key seen: 0; a NaN stays one
            T* op = static_cast<T*>(a.out) + at * D + d;
            T t[4] = {from_f32<T>(v.x * inv), from_f32<T>(v.y * inv), from_f32<T>(v.z * inv), from_f32<T>(v.w * inv)};
            if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(op) = *reinterpret_cast<const uint4*>(t);
            else *reinterpret_cast<uint2*>(op) = *reinterpret_cast<const uint2*>(t);
            if (a.lse && d == 0) {   // l may be 2^40: its power of two goes to m
                const int e = min(max((int)(__float_as_uint(ll) >> 23) - 127, -126), 126);
                a.lse[at] = ll == 0.0f ? -INFINITY
                                       : ((mm + (float)e) + log2f(ll * __uint_as_float((127 - e) << 23))) * 0.6931471805599453f;
            }
        };
        for (int i = threadIdx.x; i < rows * (D / 4); i += kThreads) {
            const int row = i / (D / 4), d = i % (D / 4) * 4;
            const float* w = results;
            float mm = -INFINITY, ll = 0.0f;
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int k = 0; k < kAttendWarps; ++k) mm = fmaxf(mm, w[k * kWarpFloats + kRows * kPitch + 2 * row]);
            const float off = mm == -INFINITY ? 0.0f : mm;
#pragma unroll
            for (int k = 0; k < kAttendWarps; ++k) {
                const float f = exp2_approx(w[k * kWarpFloats + kRows * kPitch + 2 * row] - off);
                ll = fmaf(w[k * kWarpFloats + kRows * kPitch + 2 * row + 1], f, ll);
                const float4 t = *reinterpret_cast<const float4*>(w + k * kWarpFloats + row * kPitch + d);
                v.x = fmaf(t.x, f, v.x), v.y = fmaf(t.y, f, v.y), v.z = fmaf(t.z, f, v.z), v.w = fmaf(t.w, f, v.w);
            }
            if (whole) {
                write(row, d, v, mm, ll);
            } else {
                *reinterpret_cast<float2*>(part + row * (D + 2) + d) = make_float2(v.x, v.y);
                *reinterpret_cast<float2*>(part + row * (D + 2) + d + 2) = make_float2(v.z, v.w);
                if (d == 0) *reinterpret_cast<float2*>(part + row * (D + 2) + D) = make_float2(mm, ll);
            }
        }
        if (!whole) {
            __threadfence();
            __syncthreads();
            if (threadIdx.x == 0) {   // the blocks that hold its granules
                const long long item = u0 + sg.before + kAttendItemCost;
                join_from = (int)(item / chunk);
                join_to = (int)((item + sg.n - 1) / chunk);
                is_last = atomicAdd(a.counter + join_from, 1) == join_to - join_from;
            }
            __syncthreads();
            if (is_last) {
                const long long c0 = join_from, c1 = join_to;
                __threadfence();
                if (threadIdx.x == 0) a.counter[c0] = 0;
                // The item begins in block c0 (its second part) and covers the
                // first part of every later one.
                const float* p0 = a.part + (2 * c0 + 1) * kRows * (D + 2);
                const long long step = 2ll * kRows * (D + 2);
                for (int i = threadIdx.x; i < rows * (D / 4); i += kThreads) {
                    const int row = i / (D / 4), d = i % (D / 4) * 4;
                    float mm = -INFINITY, ll = 0.0f;
                    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
                    for (long long c = c0; c <= c1; ++c) {
                        const float* p = p0 + (c - c0) * step - (c > c0 ? kRows * (D + 2) : 0) + row * (D + 2);
                        const float2 ml = __ldcg(reinterpret_cast<const float2*>(p + D));
                        const float2 x0 = __ldcg(reinterpret_cast<const float2*>(p + d));
                        const float2 x1 = __ldcg(reinterpret_cast<const float2*>(p + d + 2));
                        const float big = fmaxf(mm, ml.x), off = big == -INFINITY ? 0.0f : big;
                        const float f0 = exp2_approx(mm - off), f1 = exp2_approx(ml.x - off);
                        mm = big;
                        ll = fmaf(ll, f0, ml.y * f1);
                        v.x = fmaf(v.x, f0, x0.x * f1), v.y = fmaf(v.y, f0, x0.y * f1);
                        v.z = fmaf(v.z, f0, x1.x * f1), v.w = fmaf(v.w, f0, x1.y * f1);
                    }
                    write(row, d, v, mm, ll);
                }
            }
        }
    }
}

}  // namespace
}  // namespace moe

using namespace moe;

namespace {

// The warps' rings, then their results.
template <int D, int NT, int kPlanes> constexpr int attend_smem_bytes() {
    return kAttendWarps * (kAttendStages * 2 * kv4_granule(D) + 8 * NT / kPlanes * (D + 4 + 2) * 4);
}

template <class T, int D, int NT, int kPlanes> cudaError_t attend_attribute() {
    return cudaFuncSetAttribute(attend_kernel<T, D, NT, kPlanes>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                attend_smem_bytes<D, NT, kPlanes>());
}

template <class T, int D> cudaError_t attend_attributes_of() {
    cudaError_t e = attend_attribute<T, D, 1, 2>();
    if constexpr (sizeof(T) == 4) {
        if (e == cudaSuccess) e = attend_attribute<T, D, 2, 2>();
    } else {
        if (e == cudaSuccess) e = attend_attribute<T, D, 1, 1>();
        if (e == cudaSuccess) e = attend_attribute<T, D, 2, 1>();
    }
    return e;
}

template <int D> cudaError_t attend_attributes_dim() {
    cudaError_t e = attend_attributes_of<float, D>();
    if (e == cudaSuccess) e = attend_attributes_of<__nv_bfloat16, D>();
    if (e == cudaSuccess) e = attend_attributes_of<__half, D>();
    return e;
}

cudaError_t attend_attributes(int D) { return D == 64 ? attend_attributes_dim<64>() : attend_attributes_dim<128>(); }

}  // namespace

struct MoeKv4 {
    MoeKv4Config cfg;
    int sms = 0;
    float* part = nullptr;     // attention: partial rows of items that several blocks share
    int* counter = nullptr;    // behind them
    int* error = nullptr;      // pinned host memory: a kernel's wait ran out
    size_t bytes = 0;
};

namespace {

// The handles' error words.  Pinning memory costs milliseconds, so they share
// pages that stay the process's; a word is given back only after its device has
// no work of the handle left.
class ErrorWords {
public:
    cudaError_t take(int** out) {
        std::lock_guard<std::mutex> lock(mutex_);
        if (free_.empty()) {
            constexpr int kWords = 1024;
            free_.reserve(kWords * (pages_ + 1));    // giving one back never allocates
            int* page = nullptr;
            const cudaError_t e = cudaHostAlloc(reinterpret_cast<void**>(&page), kWords * sizeof(int),
                                                cudaHostAllocMapped | cudaHostAllocPortable);
            if (e != cudaSuccess) return e;
            ++pages_;
            for (int i = 0; i < kWords; ++i) free_.push_back(page + i);
        }
        *out = free_.back();
        free_.pop_back();
        **out = 0;
        return cudaSuccess;
    }
    void give(int* word) {
        if (!word) return;
        std::lock_guard<std::mutex> lock(mutex_);
        free_.push_back(word);
    }

private:
    std::mutex mutex_;
    std::vector<int*> free_;
    size_t pages_ = 0;
};

ErrorWords& error_words() {
    static ErrorWords* words = new ErrorWords;    // not destroyed: handles may be, at the process's end
    return *words;
}

}  // namespace

extern "C" {

void moe_kv4_config_init(MoeKv4Config* c) {
    if (!c) return;
    *c = MoeKv4Config{};
    c->num_kv_heads = 16;
    c->head_dim = 128;
    c->block_tokens = 16;
    c->table_width = 40;
    c->max_requests = 16;
    c->num_blocks = 640;
}

int moe_kv4_create(const MoeKv4Config* cfg, MoeKv4** out) {
    return guarded("moe_kv4_create", [&]() -> int {
        if (!cfg || !out) return report_error(MOE_ERR_INVALID, "moe_kv4_create: null argument");
        *out = nullptr;
        if (cfg->num_kv_heads < 1 || cfg->num_kv_heads > 256)
            return report_error(MOE_ERR_INVALID, "moe_kv4_create: num_kv_heads must be 1..256");
        if (cfg->head_dim != 64 && cfg->head_dim != 128)
            return report_error(MOE_ERR_UNSUPPORTED, "moe_kv4_create: head_dim must be 64 or 128");
        if (cfg->block_tokens < 16 || cfg->block_tokens > 1024 || cfg->block_tokens % 16)
            return report_error(MOE_ERR_INVALID, "moe_kv4_create: block_tokens must be a multiple of 16, 16..1024");
        if ((long long)cfg->num_blocks * cfg->num_kv_heads * (cfg->block_tokens / 16) >= 0xffffffffll ||
            (long long)cfg->num_blocks * (cfg->block_tokens / 16) > 0x7fffffffll)
            return report_error(MOE_ERR_UNSUPPORTED, "moe_kv4_create: a cache of 2^32 granules, or of 2^31 per head, or more");
        if (cfg->num_blocks < 1 || cfg->table_width < 1 ||
            (long long)cfg->table_width * cfg->block_tokens > (1 << 30))
            return report_error(MOE_ERR_INVALID, "moe_kv4_create: need num_blocks >= 1, table_width >= 1 and "
                                                 "table_width * block_tokens <= 2^30");
        if (cfg->max_requests < 1 || cfg->max_requests > kMaxRequests)
            return report_error(MOE_ERR_INVALID, "moe_kv4_create: max_requests must be 1..8192");
        int ndev = 0;
        if (cudaGetDeviceCount(&ndev) != cudaSuccess || cfg->device < 0 || cfg->device >= ndev)
            return report_error(MOE_ERR_INVALID, "moe_kv4_create: no such device");
        OnDevice on(cfg->device);
        int major = 0, sms = 0;
        cudaError_t e = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, cfg->device);
        if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, cfg->device);
        // The kernel's limit, not the handle's: every handle asks for the same.
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     (int)plan_smem_bytes(kMaxRequests));
        if (e == cudaSuccess) e = attend_attributes(cfg->head_dim);
        if (e != cudaSuccess) return launch_status(e, "moe_kv4_create");
        if (!on.ok) return report_error(MOE_ERR_CUDA, "moe_kv4_create: cannot select the device");
        if (major != 10)
            return report_error(MOE_ERR_UNSUPPORTED, "libmoe_b200 is built for sm_100a (B200) only");
        std::unique_ptr<MoeKv4, void (*)(MoeKv4*)> h(new MoeKv4, moe_kv4_destroy);
        h->cfg = *cfg;
        h->sms = sms;
        const size_t grid = (size_t)sms * kAttendCtasPerSm;
        const size_t part = grid * 2 * 16 * (cfg->head_dim + 2) * sizeof(float);
        const size_t counter = grid * sizeof(int);
        e = handle_alloc(cfg->device, part + counter, reinterpret_cast<void**>(&h->part));
        if (e == cudaSuccess) {
            h->counter = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(h->part) + part);
            e = cudaMemset(h->counter, 0, counter);
        }
        if (e == cudaSuccess) e = cudaDeviceSynchronize();
        if (e == cudaSuccess) e = error_words().take(&h->error);
        if (e != cudaSuccess) {
            cudaGetLastError();
            return report_error(e == cudaErrorMemoryAllocation ? MOE_ERR_OOM : MOE_ERR_CUDA,
                                std::string("moe_kv4_create: ") + cudaGetErrorString(e));
        }
        h->bytes = part + counter;
        *out = h.release();
        return MOE_OK;
    });
}

void moe_kv4_destroy(MoeKv4* h) {
    if (!h) return;
    OnDevice on(h->cfg.device);
    handle_free(h->part);     // waits for what still uses it
    error_words().give(h->error);
    delete h;
}

size_t moe_kv4_cache_bytes(const MoeKv4* h) {
    if (!h) return 0;
    const MoeKv4Config& c = h->cfg;
    return (size_t)c.num_blocks * c.num_kv_heads * (c.block_tokens / 16) * kv4_granule(c.head_dim);
}

size_t moe_kv4_device_bytes(const MoeKv4* h) { return h ? h->bytes : 0; }

int moe_kv4_plan_device(MoeKv4* h, const int32_t* cached_len, const int32_t* new_len, int32_t R, int32_t* free_ring,
                        const int32_t* ring_state, int32_t* block_table, int32_t* kv_len, int32_t* q_offset,
                        int32_t* position, int64_t* slot, int32_t tokens_cap, int32_t* ring_state_out, void* stream) {
    return guarded("moe_kv4_plan_device", [&]() -> int {
        if (!h) return report_error(MOE_ERR_INVALID, "moe_kv4_plan_device: null handle");
        const MoeKv4Config& c = h->cfg;
        if (R < 1 || R > c.max_requests || tokens_cap < 0)
            return report_error(MOE_ERR_INVALID, "moe_kv4_plan_device: need 1 <= num_requests <= max_requests and "
                                                 "tokens_cap >= 0");
        if (!cached_len || !new_len || !free_ring || !ring_state || !block_table || !kv_len || !q_offset ||
            !ring_state_out || (tokens_cap > 0 && (!position || !slot)))
            return report_error(MOE_ERR_INVALID, "moe_kv4_plan_device: null pointer argument");
        if (ring_state_out == ring_state)
            return report_error(MOE_ERR_INVALID, "moe_kv4_plan_device: ring_state_out must not be ring_state");
        if (kv_len == cached_len || kv_len == new_len)
            return report_error(MOE_ERR_INVALID, "moe_kv4_plan_device: kv_len must not be cached_len or new_len");
        OnDevice on(c.device);
        if (!on.ok) return report_error(MOE_ERR_CUDA, "moe_kv4_plan_device: cannot select the device");
        PlanArgs a{cached_len, new_len, R, c.table_width, c.block_tokens, c.num_blocks, tokens_cap, free_ring,
                   ring_state, block_table, kv_len, q_offset, position,
                   reinterpret_cast<long long*>(slot), ring_state_out, FastDiv(c.block_tokens)};
        const size_t smem = plan_smem_bytes(R);
        // A thread per token, a block for every 64 requests' rows, one block per SM at most.
        const int grid = std::max(1, std::min(h->sms, std::max(tokens_cap / kPlanThreads + 1, (R + 63) / 64)));
        return launch_status(launch(plan_kernel, grid, kPlanThreads, smem, static_cast<cudaStream_t>(stream), false, a),
                             "moe_kv4_plan_device");
    });
}

}  // extern "C"

namespace {

template <class T, int D> cudaError_t append_typed(const AppendArgs& a, bool vec, cudaStream_t s) {
    const dim3 grid((unsigned)((a.N + 15) / 16 * (long long)a.H));
    return vec ? launch(append_kernel<T, D, true>, grid, D, 0, s, false, a)
               : launch(append_kernel<T, D, false>, grid, D, 0, s, false, a);
}

template <class T> cudaError_t append_dim(const AppendArgs& a, int D, bool vec, cudaStream_t s) {
    return D == 64 ? append_typed<T, 64>(a, vec, s) : append_typed<T, 128>(a, vec, s);
}

template <class T, int D, int NT, int kPlanes> cudaError_t attend_launch(const AttendArgs& a, int sms, cudaStream_t s) {
    return launch(attend_kernel<T, D, NT, kPlanes>, sms * (NT == 1 ? kAttendCtasPerSm : 2), dim3(kAttendWarps * 32),
                  attend_smem_bytes<D, NT, kPlanes>(), s, false, a);
}

template <class T, int D> cudaError_t attend_tiles(const AttendArgs& a, int sms, cudaStream_t s) {
    // Rows that a request's queries of one key/value head have on average.  Up to 4 the 8 columns
    // of a product hold two planes of each (why at attend_kernel).
    const long long rows = (long long)(a.H / a.Hkv) * ((a.tokens + a.R - 1) / a.R);
    if (rows <= 4) return attend_launch<T, D, 1, 2>(a, sms, s);
    if constexpr (sizeof(T) == 4) return attend_launch<T, D, 2, 2>(a, sms, s);
    else return rows <= 8 ? attend_launch<T, D, 1, 1>(a, sms, s) : attend_launch<T, D, 2, 1>(a, sms, s);
}

template <class T> cudaError_t attend_dim(const AttendArgs& a, int D, int sms, cudaStream_t s) {
    return D == 64 ? attend_tiles<T, 64>(a, sms, s) : attend_tiles<T, 128>(a, sms, s);
}

}  // namespace

extern "C" {

int moe_kv4_append_device(MoeKv4* h, void* cache, const void* k, const void* v, int32_t dtype, int32_t tokens,
                          int64_t k_token_stride, int64_t k_head_stride, int64_t v_token_stride,
                          int64_t v_head_stride, const int64_t* slot, void* k_out, void* v_out, void* stream) {
    return guarded("moe_kv4_append_device", [&]() -> int {
        if (!h) return report_error(MOE_ERR_INVALID, "moe_kv4_append_device: null handle");
        const MoeKv4Config& c = h->cfg;
        if (!valid_dtype(dtype)) return report_error(MOE_ERR_INVALID, "moe_kv4_append_device: unknown dtype");
        if (tokens < 0) return report_error(MOE_ERR_INVALID, "moe_kv4_append_device: tokens must not be negative");
        if (((long long)tokens + 15) / 16 * c.num_kv_heads > 0x7fffffffll)
            return report_error(MOE_ERR_UNSUPPORTED, "moe_kv4_append_device: too many tokens for one call");
        if (tokens == 0) return MOE_OK;
        if (!cache || !k || !v || !slot)
            return report_error(MOE_ERR_INVALID, "moe_kv4_append_device: null pointer argument");
        const size_t es = dtype_bytes(dtype);
        if (!aligned16(cache) || (k_out && !aligned16(k_out)) || (v_out && !aligned16(v_out)) || !aligned_to(k, es) ||
            !aligned_to(v, es) || !aligned_to(slot, 8))
            return report_error(MOE_ERR_INVALID, "moe_kv4_append_device: cache, k_out and v_out must be 16-byte "
                                                 "aligned, k, v and slot to their elements");
        OnDevice on(c.device);
        if (!on.ok) return report_error(MOE_ERR_CUDA, "moe_kv4_append_device: cannot select the device");
        AppendArgs a{static_cast<uint8_t*>(cache), {k, v}, {k_token_stride, v_token_stride},
                     {k_head_stride, v_head_stride}, reinterpret_cast<const long long*>(slot), {k_out, v_out}, tokens,
                     c.num_kv_heads, c.block_tokens, c.num_blocks, FastDiv(c.num_kv_heads), FastDiv(c.block_tokens / 16)};
        bool vec = aligned16(k) && aligned16(v);
        for (int64_t st : {k_token_stride, k_head_stride, v_token_stride, v_head_stride})
            vec = vec && (st * (int64_t)es) % 16 == 0;
        const cudaStream_t s = static_cast<cudaStream_t>(stream);
        cudaError_t e = dtype == MOE_DTYPE_F32    ? append_dim<float>(a, c.head_dim, vec, s)
                        : dtype == MOE_DTYPE_BF16 ? append_dim<__nv_bfloat16>(a, c.head_dim, vec, s)
                                                  : append_dim<__half>(a, c.head_dim, vec, s);
        return launch_status(e, "moe_kv4_append_device");
    });
}

int moe_kv4_attention_device(MoeKv4* h, const void* cache, const void* q, int32_t dtype, int32_t tokens,
                             int32_t num_heads, int64_t q_token_stride, int64_t q_head_stride,
                             const int32_t* block_table, const int32_t* kv_len, const int32_t* q_offset, int32_t R,
                             float scale, int32_t window, void* out, float* lse, void* stream) {
    return guarded("moe_kv4_attention_device", [&]() -> int {
        if (!h) return report_error(MOE_ERR_INVALID, "moe_kv4_attention_device: null handle");
        const MoeKv4Config& c = h->cfg;
        if (!valid_dtype(dtype)) return report_error(MOE_ERR_INVALID, "moe_kv4_attention_device: unknown dtype");
        if (num_heads < 1 || num_heads % c.num_kv_heads || num_heads / c.num_kv_heads > 64)
            return report_error(MOE_ERR_INVALID, "moe_kv4_attention_device: num_heads must be a multiple of "
                                                 "num_kv_heads, at most 64 times it");
        if (R < 1 || R > c.max_requests || tokens < 0 || window < 0 || !std::isfinite(scale))
            return report_error(MOE_ERR_INVALID, "moe_kv4_attention_device: need 1 <= num_requests <= max_requests, "
                                                 "tokens >= 0, window >= 0 and a finite scale");
        if ((long long)tokens * num_heads > 0x7fffffffll || tokens > (1 << 30))
            return report_error(MOE_ERR_UNSUPPORTED, "moe_kv4_attention_device: too many tokens for one call");
        if (tokens == 0) return MOE_OK;
        if (!cache || !q || !block_table || !kv_len || !q_offset || !out)
            return report_error(MOE_ERR_INVALID, "moe_kv4_attention_device: null pointer argument");
        if (!aligned16(cache) || !aligned16(out) || !aligned_to(q, dtype_bytes(dtype)))
            return report_error(MOE_ERR_INVALID, "moe_kv4_attention_device: cache and out must be 16-byte aligned, q "
                                                 "to its elements");
        if (*static_cast<volatile int*>(h->error))
            return report_error(MOE_ERR_TIMEOUT, "moe_kv4_attention_device: a copy of an earlier call did not arrive "
                                                 "in time; its results, and this handle, are not to be used");
        OnDevice on(c.device);
        if (!on.ok) return report_error(MOE_ERR_CUDA, "moe_kv4_attention_device: cannot select the device");
        AttendArgs a{static_cast<const uint8_t*>(cache), q, q_token_stride, q_head_stride, block_table, kv_len,
                     q_offset, out, lse, h->part, h->counter, h->error, tokens, num_heads, c.num_kv_heads, R, c.table_width, c.block_tokens,
                     c.num_blocks, (long long)window >= (long long)c.table_width * c.block_tokens ? 0 : window, scale, false,
                     FastDiv(num_heads / c.num_kv_heads), FastDiv(c.block_tokens / 16)};
        const cudaStream_t s = static_cast<cudaStream_t>(stream);
        const int64_t es = (int64_t)dtype_bytes(dtype);
        a.vec = aligned16(q) && q_token_stride * es % 16 == 0 && q_head_stride * es % 16 == 0;
        cudaError_t e = dtype == MOE_DTYPE_F32    ? attend_dim<float>(a, c.head_dim, h->sms, s)
                        : dtype == MOE_DTYPE_BF16 ? attend_dim<__nv_bfloat16>(a, c.head_dim, h->sms, s)
                                                  : attend_dim<__half>(a, c.head_dim, h->sms, s);
        return launch_status(e, "moe_kv4_attention_device");
    });
}

}  // extern "C"
