// Matrix-vector products with 4-bit group-scaled weights, and the routed
// experts built on them.
#include <cstring>
#include <new>

#include "dtype.cuh"
#include "moe_internal.h"

namespace moe {
namespace {

struct W4Args {
    const uint8_t* codes;
    const __half* scales;
    const uint8_t* zeros;
    const void* x;
    const int* matrix;
    void* y;
    long long x_stride;
    int rows, x_share, E, N, K, group, outputs;
    bool gated;
};

template <class T> __device__ float row_dot(const W4Args& a, int e, int n, const T* x, int lane) {
    const long long row = (long long)e * a.N + n;
    const uint8_t* c = a.codes + row * (a.K / 2);
    const int groups = (a.K + a.group - 1) / a.group;
    float sum = 0.0f;
    for (int k = lane * 8; k < a.K; k += 256) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(c + k / 2);
        const long long g = row * groups + k / a.group;
        const float z = a.zeros ? (float)a.zeros[g] : 8.0f, s = __half2float(a.scales[g]);
        float part = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) part = fmaf((float)((w >> (4 * i)) & 15) - z, to_f32(x[k + i]), part);
        sum = fmaf(s, part, sum);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sum;
}

// One warp per output.
template <class TX, class TY> __global__ void __launch_bounds__(256) matvec_kernel(W4Args a) {
    const int lane = threadIdx.x & 31, n = blockIdx.x * 8 + (threadIdx.x >> 5), i = blockIdx.y;
    if (n >= a.outputs) return;
    const int e = a.matrix ? a.matrix[i] : 0;
    float v = 0.0f;
    if (e >= 0 && e < a.E) {
        const TX* x = static_cast<const TX*>(a.x) + (i / a.x_share) * a.x_stride;
        v = row_dot(a, e, n, x, lane);
        if (a.gated) v = v / (1.0f + expf(-v)) * row_dot(a, e, n + a.outputs, x, lane);
    }
    if (lane == 0) static_cast<TY*>(a.y)[(long long)i * a.outputs + n] = from_f32<TY>(v);
}

// y[t] = sum over s of w[t][s] * part[t * k + s], s ascending.
template <class T> __global__ void __launch_bounds__(256) experts_sum_kernel(const float* part, const int* idx, const float* w, T* y, int k, int d, int E) {
    const int n = blockIdx.x * 256 + threadIdx.x, t = blockIdx.y;
    if (n >= d) return;
    float v = 0.0f;
    for (int s = 0; s < k; ++s) {
        const int e = idx[t * k + s];
        if (e >= 0 && e < E) v = fmaf(w[t * k + s], part[((long long)t * k + s) * d + n], v);
    }
    y[(long long)t * d + n] = from_f32<T>(v);
}

constexpr int kMaxRows = 512;

}  // namespace
}  // namespace moe

using namespace moe;

struct MoeW4 {
    MoeW4Config cfg;
    int outputs = 0, groups = 0;
    uint8_t* codes = nullptr;
    __half* scales = nullptr;
    uint8_t* zeros = nullptr;
    float* work = nullptr;    // this matrix's fp32 results of the experts: [work_rows][outputs]
    int work_rows = 0;
    size_t bytes = 0;
};

namespace {

int ensure_rows(MoeW4* h, int rows) {
    if (rows <= h->work_rows) return MOE_OK;
    float* p = nullptr;
    const size_t n = (size_t)rows * h->outputs * sizeof(float);
    if (cudaMalloc(&p, n) != cudaSuccess) {
        cudaGetLastError();
        return report_error(MOE_ERR_OOM, "4-bit weights: workspace allocation failed");
    }
    cudaFree(h->work);
    h->bytes += n - (size_t)h->work_rows * h->outputs * sizeof(float);
    h->work = p;
    h->work_rows = rows;
    return MOE_OK;
}

int w4_create(const MoeW4Config* cfg, const uint8_t* codes, const void* scales, const uint8_t* zeros, MoeW4** out,
              cudaMemcpyKind kind) {
    if (!cfg || !codes || !scales || !out) return report_error(MOE_ERR_INVALID, "moe_w4_create: null argument");
    *out = nullptr;
    if (cfg->num_matrices < 1 || cfg->num_matrices > 256)
        return report_error(MOE_ERR_INVALID, "moe_w4_create: num_matrices must be 1..256");
    if (cfg->rows < 1 || (cfg->gated && cfg->rows % 2) || cfg->rows > (1 << 24))
        return report_error(MOE_ERR_INVALID, "moe_w4_create: rows must be 1..2^24, even if gated");
    if (cfg->cols < 32 || cfg->cols % 32 || cfg->cols > 65536)
        return report_error(MOE_ERR_INVALID, "moe_w4_create: cols must be a multiple of 32, 32..65536");
    if (cfg->group != 32 && cfg->group != 64 && cfg->group != 128)
        return report_error(MOE_ERR_INVALID, "moe_w4_create: group must be 32, 64 or 128");
    if (cfg->max_rows < 0 || cfg->max_rows > kMaxRows)
        return report_error(MOE_ERR_INVALID, "moe_w4_create: max_rows must be 0..512");
    int ndev = 0;
    if (cudaGetDeviceCount(&ndev) != cudaSuccess || cfg->device < 0 || cfg->device >= ndev)
        return report_error(MOE_ERR_INVALID, "moe_w4_create: no such device");
    OnDevice on(cfg->device);
    int major = 0;
    cudaError_t e = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, cfg->device);
    if (e != cudaSuccess || !on.ok) return launch_status(e, "moe_w4_create");
    if (major != 10) return report_error(MOE_ERR_UNSUPPORTED, "libmoe_b200 is built for sm_100a (B200) only");
    auto* h = new MoeW4;
    h->cfg = *cfg;
    h->outputs = cfg->gated ? cfg->rows / 2 : cfg->rows;
    h->groups = (cfg->cols + cfg->group - 1) / cfg->group;
    const size_t rows = (size_t)cfg->num_matrices * cfg->rows;
    const size_t nc = rows * (cfg->cols / 2), ng = rows * h->groups;
    e = cudaMalloc(&h->codes, nc);
    if (e == cudaSuccess) e = cudaMalloc(&h->scales, ng * 2);
    if (e == cudaSuccess && zeros) e = cudaMalloc(&h->zeros, ng);
    if (e != cudaSuccess) {
        cudaGetLastError();
        moe_w4_destroy(h);
        return report_error(MOE_ERR_OOM, "moe_w4_create: device allocation failed");
    }
    e = cudaDeviceSynchronize();   // device sources may still be written on any stream
    if (e == cudaSuccess) e = cudaMemcpy(h->codes, codes, nc, kind);
    if (e == cudaSuccess) e = cudaMemcpy(h->scales, scales, ng * 2, kind);
    if (e == cudaSuccess && zeros) e = cudaMemcpy(h->zeros, zeros, ng, kind);
    if (e == cudaSuccess) e = cudaDeviceSynchronize();
    h->bytes = nc + ng * (zeros ? 3 : 2);
    int rc = launch_status(e, "moe_w4_create");
    if (rc == MOE_OK) rc = ensure_rows(h, cfg->max_rows);
    if (rc != MOE_OK) {
        moe_w4_destroy(h);
        return rc;
    }
    *out = h;
    return MOE_OK;
}

template <class TX, class TY>
cudaError_t matvec_typed(const MoeW4* h, const void* x, int rows, int64_t x_stride, int x_share, const int* matrix,
                         void* y, cudaStream_t s) {
    W4Args a{h->codes, h->scales, h->zeros, x, matrix, y, x_stride, rows, x_share, h->cfg.num_matrices, h->cfg.rows,
             h->cfg.cols, h->cfg.group, h->outputs, h->cfg.gated != 0};
    return launch(matvec_kernel<TX, TY>, dim3((h->outputs + 7) / 8, rows), 256, 0, s, false, a);
}

template <class T>
cudaError_t experts_typed(MoeW4* gu, MoeW4* dn, const void* x, int T_, int k, const int* idx, const float* w, void* y,
                          cudaStream_t s) {
    cudaError_t e = matvec_typed<T, float>(gu, x, T_ * k, gu->cfg.cols, k, idx, gu->work, s);
    if (e == cudaSuccess) e = matvec_typed<float, float>(dn, gu->work, T_ * k, dn->cfg.cols, 1, idx, dn->work, s);
    if (e != cudaSuccess) return e;
    return launch(experts_sum_kernel<T>, dim3((dn->outputs + 255) / 256, T_), 256, 0, s, false, dn->work, idx, w,
                  static_cast<T*>(y), k, dn->outputs, dn->cfg.num_matrices);
}

}  // namespace

extern "C" {

void moe_w4_config_init(MoeW4Config* c) {
    if (!c) return;
    *c = MoeW4Config{};
    c->num_matrices = 1;
    c->rows = 4096;
    c->cols = 4096;
    c->group = 128;
    c->max_rows = 16;
}

int moe_w4_create(const MoeW4Config* cfg, const uint8_t* codes, const void* scales, const uint8_t* zeros,
                  MoeW4** out) {
    return guarded("moe_w4_create", [&] { return w4_create(cfg, codes, scales, zeros, out, cudaMemcpyHostToDevice); });
}

int moe_w4_create_from_device(const MoeW4Config* cfg, const uint8_t* codes, const void* scales, const uint8_t* zeros,
                              MoeW4** out) {
    return guarded("moe_w4_create_from_device",
                   [&] { return w4_create(cfg, codes, scales, zeros, out, cudaMemcpyDeviceToDevice); });
}

void moe_w4_destroy(MoeW4* h) {
    if (!h) return;
    OnDevice on(h->cfg.device);
    cudaFree(h->codes);
    cudaFree(h->scales);
    cudaFree(h->zeros);
    cudaFree(h->work);
    delete h;
}

size_t moe_w4_device_bytes(const MoeW4* h) { return h ? h->bytes : 0; }

int moe_w4_matvec_device(MoeW4* h, const void* x, int32_t dtype, int32_t num_rows, int64_t x_row_stride,
                         int32_t x_share, const int32_t* matrix, void* y, void* stream) {
    return guarded("moe_w4_matvec_device", [&]() -> int {
        if (!h) return report_error(MOE_ERR_INVALID, "moe_w4_matvec_device: null handle");
        if (!valid_dtype(dtype)) return report_error(MOE_ERR_INVALID, "moe_w4_matvec_device: unknown dtype");
        if (num_rows < 0 || num_rows > kMaxRows || x_share < 1)
            return report_error(MOE_ERR_INVALID, "moe_w4_matvec_device: need 0 <= num_rows <= 512 and x_share >= 1");
        if (num_rows == 0) return MOE_OK;
        if (!x || !y) return report_error(MOE_ERR_INVALID, "moe_w4_matvec_device: null pointer argument");
        if (!aligned_to(x, dtype_bytes(dtype)) || !aligned_to(y, dtype_bytes(dtype)))
            return report_error(MOE_ERR_INVALID, "moe_w4_matvec_device: x and y must be aligned to their elements");
        OnDevice on(h->cfg.device);
        if (!on.ok) return report_error(MOE_ERR_CUDA, "moe_w4_matvec_device: cannot select the device");
        const cudaStream_t s = static_cast<cudaStream_t>(stream);
        cudaError_t e;
        if (dtype == MOE_DTYPE_F32)
            e = matvec_typed<float, float>(h, x, num_rows, x_row_stride, x_share, matrix, y, s);
        else if (dtype == MOE_DTYPE_BF16)
            e = matvec_typed<__nv_bfloat16, __nv_bfloat16>(h, x, num_rows, x_row_stride, x_share, matrix, y, s);
        else
            e = matvec_typed<__half, __half>(h, x, num_rows, x_row_stride, x_share, matrix, y, s);
        return launch_status(e, "moe_w4_matvec_device");
    });
}

int moe_w4_experts_device(MoeW4* gu, MoeW4* dn, const void* x, int32_t dtype, int32_t T, int32_t top_k,
                          const int32_t* idx, const float* weights, void* y, void* stream) {
    return guarded("moe_w4_experts_device", [&]() -> int {
        if (!gu || !dn) return report_error(MOE_ERR_INVALID, "moe_w4_experts_device: null handle");
        if (!valid_dtype(dtype)) return report_error(MOE_ERR_INVALID, "moe_w4_experts_device: unknown dtype");
        if (!gu->cfg.gated || dn->cfg.gated || gu->outputs != dn->cfg.cols ||
            gu->cfg.num_matrices != dn->cfg.num_matrices || gu->cfg.device != dn->cfg.device)
            return report_error(MOE_ERR_INVALID, "moe_w4_experts_device: gate_up must be gated with down's cols as "
                                                 "outputs, down not gated, both of one device and num_matrices");
        if (T < 0 || top_k < 1 || (long long)T * top_k > kMaxRows)
            return report_error(MOE_ERR_INVALID, "moe_w4_experts_device: need num_tokens >= 0, top_k >= 1 and "
                                                 "num_tokens * top_k <= 512");
        if (T == 0) return MOE_OK;
        if (!x || !idx || !weights || !y)
            return report_error(MOE_ERR_INVALID, "moe_w4_experts_device: null pointer argument");
        if (!aligned_to(x, dtype_bytes(dtype)) || !aligned_to(y, dtype_bytes(dtype)))
            return report_error(MOE_ERR_INVALID, "moe_w4_experts_device: x and y must be aligned to their elements");
        OnDevice on(gu->cfg.device);
        if (!on.ok) return report_error(MOE_ERR_CUDA, "moe_w4_experts_device: cannot select the device");
        int rc = ensure_rows(gu, T * top_k);
        if (rc == MOE_OK) rc = ensure_rows(dn, T * top_k);
        if (rc != MOE_OK) return rc;
        const cudaStream_t s = static_cast<cudaStream_t>(stream);
        cudaError_t e = dtype == MOE_DTYPE_F32    ? experts_typed<float>(gu, dn, x, T, top_k, idx, weights, y, s)
                        : dtype == MOE_DTYPE_BF16 ? experts_typed<__nv_bfloat16>(gu, dn, x, T, top_k, idx, weights, y, s)
                                                  : experts_typed<__half>(gu, dn, x, T, top_k, idx, weights, y, s);
        return launch_status(e, "moe_w4_experts_device");
    });
}

}  // extern "C"
