// The paged 4-bit key/value cache: block tables and slot maps (plan), the
// quantising append, and attention over the cache.
#include <algorithm>
#include <cmath>
#include <new>

#include "dtype.cuh"
#include "kv4.cuh"
#include "moe_internal.h"

namespace moe {
namespace {

// ------------------------------------------------------------------- plan
// Sum of v over the threads before this one; *total the sum over all.  Every
// thread of the block calls it; `buf` holds 33 values.
__device__ long long block_scan(long long v, long long* buf, long long* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    long long inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += u;
    }
    __syncthreads();
    if (lane == 31) buf[warp] = inc;
    __syncthreads();
    if (warp == 0) {
        long long w = lane < warps ? buf[lane] : 0;
        long long s = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long u = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += u;
        }
        buf[lane] = s - w;
        if (lane == 31) buf[32] = s;
    }
    __syncthreads();
    *total = buf[32];
    return buf[warp] + inc - v;
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
};

constexpr int kPlanThreads = 1024;

// Every block scans all requests (R <= 8192 lengths, L2-resident), so that no
// block waits for another; the requests' rows and the tokens are then split
// over the blocks.  Table entries a token reads lie before the ones written
// here, and pages returned to the ring go behind the ones taken from it, so
// the blocks' reads and writes are disjoint.
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(PlanArgs a) {
    extern __shared__ int plan_smem[];
    int* q_off = plan_smem;              // [R + 1] clipped to cap
    int* first = plan_smem + a.R + 1;    // [R] first page taken from the ring; -1 rejected; or first page given back
    __shared__ long long buf[33];
    const int per = (a.R + kPlanThreads - 1) / kPlanThreads;
    const int r0 = min(a.R, (int)threadIdx.x * per), r1 = min(a.R, r0 + per);
    int head = a.state[0], count = a.state[1];
    if (head < 0 || head >= a.nb || count < 0 || count > a.nb) head = count = 0;
    const long long limit = (long long)a.W * a.bs;

    long long grow = 0, total;
    for (int r = r0; r < r1; ++r) grow += max(0, a.added[r]);
    const long long begin = block_scan(grow, buf, &total);
    const long long tokens = total;
    long long end = begin;
    long long need = 0, back = 0;
    for (int r = r0; r < r1; ++r) {
        const long long c = a.cached[r], n = a.added[r];
        q_off[r] = (int)min(end, (long long)a.cap);
        end += max(0ll, n);
        if (c < 0 || c > limit) continue;
        if (n >= 0 && c + n <= limit && (n == 0 || end <= a.cap)) need += (c + n + a.bs - 1) / a.bs - (c + a.bs - 1) / a.bs;
        if (n < 0) back += (c + a.bs - 1) / a.bs;
    }
    if (threadIdx.x == 0) q_off[a.R] = (int)min(tokens, (long long)a.cap);
    long long all;
    long long nsum = block_scan(need, buf, &all);
    long long bsum = block_scan(back, buf, &total);
    const long long given = min(total, (long long)a.nb - count);
    end = begin;
    long long taken = 0;
    for (int r = r0; r < r1; ++r) {
        const long long c = a.cached[r], n = a.added[r];
        end += max(0ll, n);
        bool ok = false;
        long long take = 0;
        first[r] = -1;
        if (c >= 0 && c <= limit) {
            if (n >= 0 && c + n <= limit && (n == 0 || end <= a.cap)) {
                take = (c + n + a.bs - 1) / a.bs - (c + a.bs - 1) / a.bs;
                ok = take == 0 || nsum + take <= count;
                if (ok) {
                    first[r] = (int)min(nsum, (long long)count);
                    taken += take;
                }
                nsum += take;
            } else if (n < 0) {
                first[r] = (int)min(bsum, given);
                bsum += (c + a.bs - 1) / a.bs;
            }
        }
        if (blockIdx.x == 0) {
            a.kv_len[r] = ok ? (int)(c + n) : 0;
            a.q_offset[r] = q_off[r];
        }
    }
    block_scan(taken, buf, &total);
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        a.q_offset[a.R] = q_off[a.R];
        a.state_out[0] = (int)((head + total) % a.nb);
        a.state_out[1] = (int)(count - total + given);
    }
    __syncthreads();

    // The requests' rows: a warp each.
    const int lane = threadIdx.x & 31;
    const int warps = gridDim.x * (kPlanThreads / 32);
    for (int r = blockIdx.x * (kPlanThreads / 32) + (threadIdx.x >> 5); r < a.R; r += warps) {
        const int f = first[r];
        if (f < 0) continue;
        const long long c = a.cached[r], n = a.added[r];
        const long long used = (c + a.bs - 1) / a.bs;
        int* row = a.table + (size_t)r * a.W;
        if (n < 0) {
            for (long long i = lane; i < used && f + i < given; i += 32)
                a.ring[((long long)head + count + f + i) % a.nb] = row[i];
        } else {
            const long long take = (c + n + a.bs - 1) / a.bs - used;
            for (long long i = lane; i < take; i += 32) row[used + i] = a.ring[((long long)head + f + i) % a.nb];
        }
    }
    // The tokens: a thread each.
    for (int t = blockIdx.x * kPlanThreads + threadIdx.x; t < a.cap; t += gridDim.x * kPlanThreads) {
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
                const int used = (int)(((long long)c + a.bs - 1) / a.bs), b = pos / a.bs;
                const int page = b < used ? a.table[(size_t)lo * a.W + b]
                                          : a.ring[((long long)head + first[lo] + b - used) % a.nb];
                if (page >= 0 && page < a.nb) slot = (long long)page * a.bs + pos % a.bs;
            }
        }
        a.position[t] = pos;
        a.slot[t] = slot;
    }
}

// ----------------------------------------------------------------- append
// Eight consecutive elements as fp32; kVec: one or two 16-byte loads (the
// address is 16-byte aligned), else element by element.
template <class T, bool kVec> __device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
    if constexpr (kVec) {
        constexpr int kN = 16 / sizeof(T);
        T v[8];
#pragma unroll
        for (int i = 0; i < 8 / kN; ++i)
            *reinterpret_cast<uint4*>(v + i * kN) = __ldg(reinterpret_cast<const uint4*>(p) + i);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_f32(v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_f32(p[i]);
    }
}

struct AppendArgs {
    uint8_t* cache;
    const void* x[2];            // k, v
    long long token_stride[2], head_stride[2];
    const long long* slot;
    void* out[2];
    int N, H, bs, nb;
};

// One thread per 8 dims, 8 threads per group of 64, so a group's range is
// three shuffles.  blockIdx.y: 0 keys, 1 values.
template <class T, int D, bool kVec> __global__ void __launch_bounds__(256) append_kernel(AppendArgs a) {
    constexpr int G = D / 64, kThreads = D / 8;   // threads per (token, head)
    const int kv = blockIdx.y;
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    const long long th = i / kThreads;            // token * H + head
    const int m = (int)(i % kThreads);            // which 8 dims
    const bool live = th < (long long)a.N * a.H;
    const int token = live ? (int)(th / a.H) : 0, head = live ? (int)(th % a.H) : 0;
    float x[8];
    if (live) {
        load8<T, kVec>(static_cast<const T*>(a.x[kv]) + token * a.token_stride[kv] + head * a.head_stride[kv] + m * 8, x);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = 0.0f;
    }
    bool nan = false;
    float lo = 65504.0f, hi = -65504.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        nan |= x[e] != x[e];
        x[e] = fminf(fmaxf(x[e], -65504.0f), 65504.0f);
        lo = fminf(lo, x[e]);
        hi = fmaxf(hi, x[e]);
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    const unsigned nans = __ballot_sync(0xffffffffu, nan) >> ((threadIdx.x & 31) & ~7);
    __half s = __float2half_rn(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f)), z = __float2half_rn(lo);
    if (nans & 0xff) s = z = __ushort_as_half(0x7fff);
    const float sf = __half2float(s), zf = __half2float(z);
    uint32_t word = 0;
    float val[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float q = sf > 0.0f ? rintf(__fdiv_rn(__fsub_rn(x[e], zf), sf)) : 0.0f;
        const float c = fminf(fmaxf(q, 0.0f), 15.0f);
        word |= (uint32_t)c << (4 * e);
        val[e] = __fmaf_rn(sf, c, zf);   // s * c is exact in fp32
    }
    if (!live) return;
    if (a.out[kv]) {
        T* o = static_cast<T*>(a.out[kv]) + th * D + m * 8;
        T v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = from_f32<T>(val[e]);
#pragma unroll
        for (int e = 0; e < 8; e += 16 / (int)sizeof(T))
            *reinterpret_cast<uint4*>(o + e) = *reinterpret_cast<const uint4*>(v + e);
    }
    const long long slot = a.slot[token];
    if (slot < 0 || slot >= (long long)a.nb * a.bs) return;
    const long long page = slot / a.bs;
    const int off = (int)(slot % a.bs), t = off & 15, g = m >> 3;
    uint8_t* gran = a.cache + ((page * a.H + head) * (a.bs >> 4) + (off >> 4)) * kv4_granule(D);
    if (kv == 0) {
        *reinterpret_cast<uint32_t*>(gran + kv4_k_word<D>(t, m)) = word;
    } else {
        *reinterpret_cast<uint32_t*>(gran + kv4_v_word<D>(t, m)) = word;
    }
    if ((m & 7) == 0)
        *reinterpret_cast<__half2*>(gran + 16 * D + (kv * 16 + t) * G * 4 + g * 4) = __halves2half2(s, z);
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
    int tokens, H, Hkv, R, W, bs, nb, window;
    float scale;
};

// One warp per (query token, head): the keys one after the other, each lane
// owning 8 dims of every 256.
template <class T, int D> __global__ void __launch_bounds__(128) attend_kernel(AttendArgs a) {
    constexpr int kLanes = D / 8, G = D / 64;
    const int lane = threadIdx.x & 31;
    const long long w = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int token = (int)(w / a.H), head = (int)(w % a.H);
    if (token >= a.tokens) return;
    int lo = 0, hi = a.R;   // the first r with q_offset[r + 1] > token, or R
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (a.q_offset[mid + 1] > token) hi = mid;
        else lo = mid + 1;
    }
    if (lo == a.R || token < a.q_offset[lo]) return;
    const int r = lo;
    const int len = (int)min((long long)max(a.kv_len[r], 0), (long long)a.W * a.bs);
    const int pos = len - min(a.q_offset[r + 1], a.tokens) + token;
    const int kvh = head / (a.H / a.Hkv);
    const int m = lane % kLanes, g = m >> 3;
    float q[8], o[8];
    const T* qp = static_cast<const T*>(a.q) + token * a.q_token_stride + head * a.q_head_stride + m * 8;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        q[e] = to_f32(qp[e]) * a.scale;
        o[e] = 0.0f;
    }
    float mx = -INFINITY, sum = 0.0f;
    for (int t = a.window > 0 ? max(0, pos - a.window + 1) : 0; t <= pos; ++t) {
        const int page = a.table[(size_t)r * a.W + t / a.bs];
        if (page < 0 || page >= a.nb) continue;
        const int off = t % a.bs, tt = off & 15;
        const uint8_t* gran = a.cache + (((long long)page * a.Hkv + kvh) * (a.bs >> 4) + (off >> 4)) * kv4_granule(D);
        const uint32_t kw = *reinterpret_cast<const uint32_t*>(gran + kv4_k_word<D>(tt, m));
        const uint32_t vw = *reinterpret_cast<const uint32_t*>(gran + kv4_v_word<D>(tt, m));
        const float2 kp = __half22float2(*reinterpret_cast<const __half2*>(gran + 16 * D + tt * G * 4 + g * 4));
        const float2 vp = __half22float2(*reinterpret_cast<const __half2*>(gran + 16 * D + (16 + tt) * G * 4 + g * 4));
        float x = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) x += q[e] * fmaf(kp.x, (float)((kw >> (4 * e)) & 15), kp.y);
#pragma unroll
        for (int s = 1; s < kLanes; s <<= 1) x += __shfl_xor_sync(0xffffffffu, x, s);
        const float next = fmaxf(mx, x);
        const float keep = next == -INFINITY ? 1.0f : expf(mx - next), p = next == -INFINITY ? 0.0f : expf(x - next);
        mx = next;
        sum = sum * keep + p;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = o[e] * keep + p * fmaf(vp.x, (float)((vw >> (4 * e)) & 15), vp.y);
    }
    if (lane < kLanes) {
        T* op = static_cast<T*>(a.out) + ((long long)token * a.H + head) * D + m * 8;
#pragma unroll
        for (int e = 0; e < 8; ++e) op[e] = from_f32<T>(sum == 0.0f ? 0.0f : o[e] / sum);   // a NaN stays one
    }
    if (lane == 0 && a.lse) a.lse[(long long)token * a.H + head] = sum == 0.0f ? -INFINITY : mx + logf(sum);
}

}  // namespace
}  // namespace moe

struct MoeKv4 {
    MoeKv4Config cfg;
    int sm_count = 148;
};

using namespace moe;

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
        if (cfg->num_blocks < 1 || cfg->table_width < 1 ||
            (long long)cfg->table_width * cfg->block_tokens > 0x7fffffffll)
            return report_error(MOE_ERR_INVALID, "moe_kv4_create: need num_blocks >= 1, table_width >= 1 and "
                                                 "table_width * block_tokens within 31 bits");
        if (cfg->max_requests < 1 || cfg->max_requests > 8192)
            return report_error(MOE_ERR_INVALID, "moe_kv4_create: max_requests must be 1..8192");
        int ndev = 0;
        if (cudaGetDeviceCount(&ndev) != cudaSuccess || cfg->device < 0 || cfg->device >= ndev)
            return report_error(MOE_ERR_INVALID, "moe_kv4_create: no such device");
        OnDevice on(cfg->device);
        int major = 0, sms = 0;
        cudaError_t e = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, cfg->device);
        if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, cfg->device);
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     (2 * cfg->max_requests + 1) * (int)sizeof(int));
        if (e != cudaSuccess) return launch_status(e, "moe_kv4_create");
        if (!on.ok) return report_error(MOE_ERR_CUDA, "moe_kv4_create: cannot select the device");
        if (major != 10)
            return report_error(MOE_ERR_UNSUPPORTED, "libmoe_b200 is built for sm_100a (B200) only");
        auto* h = new MoeKv4;
        h->cfg = *cfg;
        h->sm_count = sms;
        *out = h;
        return MOE_OK;
    });
}

void moe_kv4_destroy(MoeKv4* h) { delete h; }

size_t moe_kv4_cache_bytes(const MoeKv4* h) {
    if (!h) return 0;
    const MoeKv4Config& c = h->cfg;
    return (size_t)c.num_blocks * c.num_kv_heads * (c.block_tokens / 16) * kv4_granule(c.head_dim);
}

size_t moe_kv4_device_bytes(const MoeKv4* h) { (void)h; return 0; }

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
        OnDevice on(c.device);
        if (!on.ok) return report_error(MOE_ERR_CUDA, "moe_kv4_plan_device: cannot select the device");
        PlanArgs a{cached_len, new_len, R, c.table_width, c.block_tokens, c.num_blocks, tokens_cap, free_ring,
                   ring_state, block_table, kv_len, q_offset, position,
                   reinterpret_cast<long long*>(slot), ring_state_out};
        const size_t smem = (size_t)(2 * R + 1) * sizeof(int);
        return launch_status(launch(plan_kernel, 1, kPlanThreads, smem, static_cast<cudaStream_t>(stream), false, a),
                             "moe_kv4_plan_device");
    });
}

}  // extern "C"

namespace {

template <class T, int D> cudaError_t append_typed(const AppendArgs& a, bool vec, cudaStream_t s) {
    const long long threads = (long long)a.N * a.H * (D / 8);
    const dim3 grid((unsigned)((threads + 255) / 256), 2);
    return vec ? launch(append_kernel<T, D, true>, grid, 256, 0, s, false, a)
               : launch(append_kernel<T, D, false>, grid, 256, 0, s, false, a);
}

template <class T> cudaError_t append_dim(const AppendArgs& a, int D, bool vec, cudaStream_t s) {
    return D == 64 ? append_typed<T, 64>(a, vec, s) : append_typed<T, 128>(a, vec, s);
}

template <class T> cudaError_t attend_dim(const AttendArgs& a, int D, cudaStream_t s) {
    const unsigned grid = (unsigned)(((long long)a.tokens * a.H + 3) / 4);
    return D == 64 ? launch(attend_kernel<T, 64>, grid, 128, 0, s, false, a)
                   : launch(attend_kernel<T, 128>, grid, 128, 0, s, false, a);
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
        if ((long long)tokens * c.num_kv_heads * (c.head_dim / 8) > 0x7fffffffll * 128)
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
                     c.num_kv_heads, c.block_tokens, c.num_blocks};
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
        if ((long long)tokens * num_heads > 0x7fffffffll)
            return report_error(MOE_ERR_UNSUPPORTED, "moe_kv4_attention_device: too many tokens for one call");
        if (tokens == 0) return MOE_OK;
        if (!cache || !q || !block_table || !kv_len || !q_offset || !out)
            return report_error(MOE_ERR_INVALID, "moe_kv4_attention_device: null pointer argument");
        if (!aligned16(cache) || !aligned16(out) || !aligned_to(q, dtype_bytes(dtype)))
            return report_error(MOE_ERR_INVALID, "moe_kv4_attention_device: cache and out must be 16-byte aligned, q "
                                                 "to its elements");
        OnDevice on(c.device);
        if (!on.ok) return report_error(MOE_ERR_CUDA, "moe_kv4_attention_device: cannot select the device");
        AttendArgs a{static_cast<const uint8_t*>(cache), q, q_token_stride, q_head_stride, block_table, kv_len,
                     q_offset, out, lse, tokens, num_heads, c.num_kv_heads, R, c.table_width, c.block_tokens,
                     c.num_blocks, window, scale};
        const cudaStream_t s = static_cast<cudaStream_t>(stream);
        cudaError_t e = dtype == MOE_DTYPE_F32    ? attend_dim<float>(a, c.head_dim, s)
                        : dtype == MOE_DTYPE_BF16 ? attend_dim<__nv_bfloat16>(a, c.head_dim, s)
                                                  : attend_dim<__half>(a, c.head_dim, s);
        return launch_status(e, "moe_kv4_attention_device");
    });
}

}  // extern "C"
