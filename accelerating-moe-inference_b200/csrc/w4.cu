// Matrix-vector products with 4-bit group-scaled weights, and the routed
// experts built on them.
#include <algorithm>
#include <memory>
#include <type_traits>
#include <new>
#include <vector>

#include "dtype.cuh"
#include "mma.cuh"
#include "moe_internal.h"
#include "ptx.cuh"

namespace moe {
namespace {

constexpr int kMaxRows = 512;        // products of one call
constexpr int kBlockK = 128;         // columns of a record
constexpr int kMaxMatrices = 256;
// What a thread block makes operands of for itself: columns of x's rows times
// blocks of 128 inputs, and bytes (two thread blocks stay on an SM).
constexpr int kInlineBlocks = 64, kInlineMax = 49152;
// Threads of a block and blocks of an SM, by tiles of rows and columns: what
// the registers allow.
__host__ __device__ constexpr int w4_threads(int NT) { return NT == 1 ? 256 : 128; }
__host__ __device__ constexpr int w4_blocks(int MT, int NT) { return NT == 1 ? 2 : MT == 1 ? 4 : 3; }

// The handle's own layout of the weights: records of 16 rows x 128 columns,
// [matrix][quad of tiles of 16 rows][block of 128 columns][4 tiles].  Lane
// 4 g + j of a warp owns, of rows g and g + 8, the columns 32 w + 8 j .. + 7 of
// each w < 4:
//   codes   [row half][lane][4 w] 32-bit words, the lowest nibble first
//   params  [8 g][row half][128 / group] (scale, zero) float16 pairs
// so that a warp reads a record with whole 512-byte loads and each lane has
// the operands of m16n8k16 products in its own registers.  A gated matrix has
// tile 2 i from the gate rows and tile 2 i + 1 from the same up rows.  Rows
// and columns of the padding have scale 0.
__host__ __device__ constexpr int w4_record(int groups) { return 1024 + 64 * groups; }

struct PackArgs {
    const uint8_t* codes;
    const __half* scales;
    const uint8_t* zeros;
    uint8_t* out;
    int rows, cols, group, tiles, blocks;
    bool gated;
};

// One block per record of one matrix; thread = (half, lane, half word pair).
__global__ void __launch_bounds__(256) w4_pack_kernel(PackArgs a) {
    const int block = blockIdx.x % a.blocks, tile = blockIdx.x / a.blocks, per = kBlockK / a.group;
    const long long matrix = blockIdx.y;
    uint8_t* rec = a.out + ((matrix * (a.tiles / 4) + tile / 4) * a.blocks + block) * (4 * w4_record(per)) + tile % 4 * w4_record(per);
    const int half_rows = a.gated ? a.rows / 2 : a.rows;
    auto row_of = [&](int r) {      // source row of the tile's row r, -1 for padding
        const int at = (a.gated ? tile >> 1 : tile) * 16 + r;
        return at < half_rows ? at + (a.gated && (tile & 1) ? half_rows : 0) : -1;
    };
    {
        const int w = threadIdx.x & 3, lane = threadIdx.x >> 2 & 31, half = threadIdx.x >> 7;
        const int row = row_of((lane >> 2) + 8 * half), k = block * kBlockK + 32 * w + 8 * (lane & 3);
        uint32_t v = 0;
        if (row >= 0 && k < a.cols)
            v = *reinterpret_cast<const uint32_t*>(a.codes + (matrix * a.rows + row) * (a.cols / 2) + k / 2);
        reinterpret_cast<uint32_t*>(rec)[threadIdx.x] = v;
    }
    if (threadIdx.x < 16 * per) {
        const int q = threadIdx.x % per, half = threadIdx.x / per & 1, g = threadIdx.x / per / 2;
        const int row = row_of(g + 8 * half), k = block * kBlockK + q * a.group;
        const int groups = (a.cols + a.group - 1) / a.group;
        __half s = __float2half_rn(0.0f), z = s;
        if (row >= 0 && k < a.cols) {
            const long long at = (matrix * a.rows + row) * groups + k / a.group;
            s = a.scales[at];
            z = __float2half_rn(a.zeros ? (float)a.zeros[at] : 8.0f);
        }
        reinterpret_cast<__half2*>(rec + 1024)[threadIdx.x] = __halves2half2(s, z);
    }
}

// Which products ask for which matrix: the matrices in use in ascending order,
// each with its products in ascending order.  A matrix's products fill column
// tiles of 8, kPlanes columns each.
struct Sorted {
    short rows[kMaxRows];           // products, sorted by matrix
    short first[kMaxMatrices + 1];  // [used + 1] into rows
    short matrix[kMaxMatrices];     // [used]
    short of[kMaxRows];             // matrix of each product, -1 outside the range
    short tile[kMaxMatrices + 1];   // [used + 1] first column tile
    short column[kMaxRows];         // first column of each product, over all column tiles
    short count[kMaxMatrices], place[kMaxMatrices];
    int used;
};

// Called by all threads of the block.
template <int kThreads, int kPlanes> __device__ void sort_products(Sorted& s, const int* matrix, int n, int E) {
    if (!matrix) {
        for (int i = threadIdx.x; i < n; i += kThreads) {
            s.rows[i] = (short)i;
            s.column[i] = (short)(i * kPlanes);
        }
        if (threadIdx.x == 0) {
            s.used = 1;
            s.matrix[0] = s.first[0] = s.tile[0] = 0;
            s.first[1] = (short)n;
            s.tile[1] = (short)((n * kPlanes + 7) / 8);
        }
        __syncthreads();
        return;
    }
    if (n <= 32) {       // one warp, a product a lane
        if (threadIdx.x < 32) {
            const int lane = threadIdx.x;
            int e = lane < n ? __ldg(matrix + lane) : -1;
            if (e >= E) e = -1;
            const bool in = e >= 0;
            const unsigned same = __match_any_sync(0xffffffffu, in ? e : -1), below = (1u << lane) - 1;
            const int rank = __popc(same & below), count = __popc(same);
            const bool leads = in && rank == 0;
            int place = 0, first = 0, tile = 0, tiles_all = 0, all = 0;   // over the matrices before this one
            for (int k = 0; k < n; ++k) {
                const int other = __shfl_sync(0xffffffffu, leads ? e : -1, k), c = __shfl_sync(0xffffffffu, count, k);
                const int t = (c * kPlanes + 7) / 8;
                if (other < 0) continue;
                all += c;
                tiles_all += t;
                if (other < e) ++place, first += c, tile += t;
            }
            const int used = __popc(__ballot_sync(0xffffffffu, leads));
            if (lane < n) s.of[lane] = (short)(in ? e : -1);
            if (in) {
                s.rows[first + rank] = (short)lane;
                s.column[lane] = (short)(tile * 8 + rank * kPlanes);
            }
            if (leads) {
                s.matrix[place] = (short)e;
                s.first[place] = (short)first;
                s.tile[place] = (short)tile;
            }
            if (lane == 0) {
                s.used = used;
                s.first[used] = (short)all;
                s.tile[used] = (short)tiles_all;
            }
        }
        __syncthreads();
        return;
    }
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const int e = __ldg(matrix + i);
        s.of[i] = (short)(e >= 0 && e < E ? e : -1);
    }
    for (int e = threadIdx.x; e < E; e += kThreads) s.count[e] = 0;
    __syncthreads();
    if (threadIdx.x < 32) {
        // Each product's place among its matrix's, 32 products at a time.
        for (int i0 = 0; i0 < n; i0 += 32) {
            const int i = i0 + threadIdx.x, e = i < n ? s.of[i] : -1;
            const unsigned same = __match_any_sync(0xffffffffu, e);
            const int rank = __popc(same & ((1u << threadIdx.x) - 1)), before = e >= 0 ? s.count[e] : 0;
            __syncwarp();
            if (e >= 0) {
                s.column[i] = (short)(before + rank);
                if (rank == 0) s.count[e] = (short)(before + __popc(same));
            }
            __syncwarp();
        }
        int used = 0, at = 0, tiles = 0;
        for (int e0 = 0; e0 < E; e0 += 32) {
            const int e = e0 + threadIdx.x, c = e < E ? s.count[e] : 0;
            const int t = (c * kPlanes + 7) / 8;
            int sum = c, tile = t;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, sum, o), u = __shfl_up_sync(0xffffffffu, tile, o);
                if (threadIdx.x >= o) sum += v, tile += u;
            }
            const unsigned m = __ballot_sync(0xffffffffu, c > 0);
            if (c > 0) {
                const int k = used + __popc(m & ((1u << threadIdx.x) - 1));
                s.matrix[k] = (short)e;
                s.first[k] = (short)(at + sum - c);
                s.tile[k] = (short)(tiles + tile - t);
                s.place[e] = (short)k;
                s.count[e] = (short)(at + sum - c);     // from here on the place of its first product
            }
            used += __popc(m);
            at += __shfl_sync(0xffffffffu, sum, 31);
            tiles += __shfl_sync(0xffffffffu, tile, 31);
        }
        if (threadIdx.x == 0) {
            s.used = used;
            s.first[used] = (short)at;
            s.tile[used] = (short)tiles;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const int e = s.of[i];
        if (e < 0) continue;
        const int rank = s.column[i];
        s.rows[s.count[e] + rank] = (short)i;
        s.column[i] = (short)(s.tile[s.place[e]] * 8 + rank * kPlanes);
    }
    __syncthreads();
}

// ------------------------------------------------------------ activations
// The activations as the products' operand B: a row of x scaled by a power of
// two to below 2^11, as one column (16-bit types: exact down to 2^-34 of the
// row's largest) or two, hi and (x - hi) 2^11 (fp32: 22 bits).  The columns of
// a matrix's products lie together, in tiles of 8, as the lanes hold them:
//   plane   [column tile][block of 128][4 w][8 columns][4 j] 16 bytes: the
//           float16 pairs (i, i + 4), i < 4, of inputs 32 w + 8 j .. + 7; with
//           one plane those of even i times 16 to match their codes' 2^-24
//   sums    [column tile][block of 128][128 / group][8 columns] of the scaled
//           values, times 2^-20
//   unit    [row of x] what a scaled sum is multiplied by
struct Planes {
    uint4* plane;
    float* sums;
    float* unit;
};

struct PlanesArgs {
    const void* x;
    long long stride;
    const int* matrix;
    Planes out;
    int cols, blocks, group, num_rows, share, E;
    bool vec;              // rows of x can be read 16 bytes at a time
    int dtype;             // of x
};

// Eight inputs of a row from `k` on, zeros past its end.
template <class T> __device__ __forceinline__ void load_chunk(const T* row, int k, int cols, bool vec, float (&v)[8]) {
    if (k >= cols) {       // cols is a multiple of 32
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    } else if (vec) {
        T t[8];
#pragma unroll
        for (int i = 0; i < 8 * (int)sizeof(T) / 16; ++i)
            *reinterpret_cast<uint4*>(t + i * (16 / sizeof(T))) = reinterpret_cast<const uint4*>(row + k)[i];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = to_f32(t[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = to_f32(row[k + i]);
    }
}

// The lanes of chunk c's warp whose chunks a row of `chunks` has, where lanes
// hold neighbouring chunks: chunks is a multiple of 16, so all or the lower half.
__device__ __forceinline__ unsigned chunk_lanes(int c, int chunks) {
    return chunks - (c & ~31) >= 32 ? 0xffffffffu : 0xffffu;
}

__device__ __forceinline__ float chunk_max(const float (&v)[8]) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(v[i]));
    return m;
}

// Exponent of a row's largest, kept where 2^(10 - e) is a normal number, the
// factor 2^(10 - e) that scales the row and its inverse.  A row that holds an
// infinity has an infinite unit (see defined_product).
struct RowScale {
    float up, unit;
    __device__ explicit RowScale(float largest) {
        const int e = min(max((int)(__float_as_uint(largest) >> 23), 11), 253);
        up = __uint_as_float((264 - e) << 23);
        unit = isinf(largest) ? largest : __uint_as_float((e - 10) << 23);
    }
};

// A scaled chunk's operands.
template <int kPlanes> __device__ __forceinline__ void operands(const float (&v)[8], uint4 (&out)[kPlanes]) {
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float f = kPlanes == 2 || (i & 1) ? 1.0f : 16.0f;
        const __half2 h = __floats2half2_rn(v[i] * f, v[i + 4] * f);
        hi[i] = *reinterpret_cast<const uint32_t*>(&h);
        if constexpr (kPlanes == 2) {
            const float2 b = __half22float2(h);
            const __half2 l = __floats2half2_rn((v[i] - b.x) * 2048.0f, (v[i + 4] - b.y) * 2048.0f);
            lo[i] = *reinterpret_cast<const uint32_t*>(&l);
        }
    }
    out[0] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    if constexpr (kPlanes == 2) out[1] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
}

// One block per row of x.  Latency is all (about 4 us, beneath the weights'
// first loads): the row is read once, all its loads at a time, and kept in
// registers (up to 16384 inputs; what is past them is read again).
template <class T, int kPlanes> __global__ void __launch_bounds__(1024) w4_planes_kernel(PlanesArgs a) {
    constexpr int kHold = 2;
    __shared__ float best[32];
    __shared__ Sorted sorted;
    const int row = blockIdx.x;
    const T* p = static_cast<const T*>(a.x) + row * a.stride;
    wait_predecessor_grid();
    launch_dependents();
    const int chunks = a.blocks * (kBlockK / 8), per = a.group / 8;
    float held[kHold][8], mx = 0.0f;
#pragma unroll
    for (int h = 0; h < kHold; ++h) load_chunk(p, (threadIdx.x + 1024 * h) * 8, a.cols, a.vec, held[h]);
    sort_products<1024, kPlanes>(sorted, a.matrix, a.num_rows, a.E);
#pragma unroll
    for (int h = 0; h < kHold; ++h) mx = fmaxf(mx, chunk_max(held[h]));
    for (int c = threadIdx.x + 1024 * kHold; c < chunks; c += 1024) {
        float v[8];
        load_chunk(p, c * 8, a.cols, a.vec, v);
        mx = fmaxf(mx, chunk_max(v));
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if ((threadIdx.x & 31) == 0) best[threadIdx.x >> 5] = mx;
    __syncthreads();
    mx = best[threadIdx.x & 31];
#pragma unroll
    for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    const RowScale scale(mx);
    if (threadIdx.x == 0) a.out.unit[row] = scale.unit;
    const int first = row * a.share, last = min(a.num_rows, first + a.share);
    auto put = [&](int c, float (&v)[8]) {     // by all of chunk_lanes(): whole groups of lanes
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += v[i] *= scale.up;
        const unsigned live = chunk_lanes(c, chunks);
        for (int o = 1; o < per; o <<= 1) sum += __shfl_xor_sync(live, sum, o);
        uint4 b[kPlanes];
        operands<kPlanes>(v, b);
        for (int i = first; i < last; ++i) {   // the products that share the row
            if (a.matrix && sorted.of[i] < 0) continue;
            const int column = sorted.column[i], block = c / 16;
            const long long at = (long long)(column / 8) * a.blocks + block;
            uint4* to = a.out.plane + at * 128 + c % 16 / 4 * 32 + column % 8 * 4 + c % 4;
#pragma unroll
            for (int k = 0; k < kPlanes; ++k) to[4 * k] = b[k];
            if (kPlanes == 1 && c % per == 0)
                a.out.sums[(at * (kBlockK / a.group) + c % 16 / per) * 8 + column % 8] = sum * (1.0f / 1048576.0f);
        }
    };
#pragma unroll
    for (int h = 0; h < kHold; ++h) {
        const int c = threadIdx.x + 1024 * h;
        if (c < chunks) put(c, held[h]);
    }
    for (int c = threadIdx.x + 1024 * kHold; c < chunks; c += 1024) {
        float v[8];
        load_chunk(p, c * 8, a.cols, a.vec, v);
        put(c, v);
    }
}

// --------------------------------------------------------------- products
struct MatvecArgs {
    const uint8_t* records;
    Planes x;
    const int* matrix;      // [num_rows], or null
    void* y;                // [num_rows][outputs]
    int num_rows, E, tiles, blocks, outputs, dtype;
    FastDiv x_share, groups;   // groups: items of a matrix
    bool gated;
    int tiles_used;         // tiles with rows of the matrix
    int groups_part, blocks_part;   // items and blocks of 128 columns of one part; a second part's sums lie num_rows on in y
};

__device__ __forceinline__ uint4 load_stream(const uint4* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.L2::128B.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

__device__ __forceinline__ void store_as(void* y, long long at, float v, int dtype) {
    if (dtype == MOE_DTYPE_F32) static_cast<float*>(y)[at] = v;
    else if (dtype == MOE_DTYPE_BF16) static_cast<__nv_bfloat16*>(y)[at] = from_f32<__nv_bfloat16>(v);
    else static_cast<__half*>(y)[at] = from_f32<__half>(v);
}

// Rows of x that hold an infinity.  Codes that are counted from their zeros only
// behind the sum, or planes whose second holds what the first leaves, would make
// NaN where an infinity of the weight's sign is due, so such a row's products are
// made by the definition, term by term: slow, behind the hot loop, and inlined,
// since calls cost the short products time (experts_one 13.85 us, 13.6 without).
__device__ __forceinline__ float load_as(const void* x, int dtype, int k) {
    return dtype == MOE_DTYPE_F32    ? static_cast<const float*>(x)[k]
           : dtype == MOE_DTYPE_BF16 ? to_f32(static_cast<const __nv_bfloat16*>(x)[k])
                                     : to_f32(static_cast<const __half*>(x)[k]);
}

__device__ __forceinline__ bool has_infinity(const void* x, int dtype, int cols) {
#pragma unroll 1
    for (int k = 0; k < cols; ++k)
        if (isinf(load_as(x, dtype, k))) return true;
    return false;
}

// Over the blocks of 128 columns [kb, kb_end); `rec` is the record of the weight
// row's tile at column block 0, `row` its row.
template <int kPer>
__device__ __forceinline__ float defined_product(const uint8_t* rec, int row, int kb, int kb_end, const void* x, int dtype, int cols) {
    float sum = 0.0f;
#pragma unroll 1
    for (; kb < kb_end; ++kb) {
        const uint8_t* at = rec + (long long)kb * (4 * w4_record(kPer));
#pragma unroll 1
        for (int i = 0; i < kBlockK / 8 && kb * kBlockK + i * 8 < cols; ++i) {      // word i / 4 of lane 4 (row % 8) + i % 4
            const uint32_t word = reinterpret_cast<const uint32_t*>(at)[(row / 8 * 32 + row % 8 * 4 + i % 4) * 4 + i / 4];
            const float2 p = __half22float2(reinterpret_cast<const __half2*>(at + 1024)[(row % 8 * 2 + row / 8) * kPer + i * kPer / 16]);
#pragma unroll 1
            for (int n = 0; n < 8; ++n)
                sum = fmaf(p.x * ((float)(word >> (4 * n) & 15) - p.y), load_as(x, dtype, kb * kBlockK + i * 8 + n), sum);
        }
    }
    return sum;
}

// An output: the row's product, or silu of a gate row's times that of the up row
// in the next tile.
template <int kPer>
__device__ __forceinline__ float defined_output(const uint8_t* rec, int row, bool gated, int kb, int kb_end, const void* x, int dtype,
                                             int cols) {
    const float v = defined_product<kPer>(rec, row, kb, kb_end, x, dtype, cols);
    return gated ? v / (1.0f + expf(-v)) * defined_product<kPer>(rec + w4_record(kPer), row, kb, kb_end, x, dtype, cols) : v;
}

// y = W x.  An item is (matrix in use, part of the columns, MT tiles of 16
// weight rows); the thread blocks take the items in turn, a warp every
// kWarps-th block of 128 columns.  One part is all columns; two, for results
// that are added up anyway, even out the last turn.
//
// Bound by reading the weights, so a warp streams its records straight into
// registers, two to four of them ahead (the first ones before the activations'
// kernel has ended, the next item's before this one's sums are joined), and no
// weight passes through shared memory.  Products: m16n8k16 with the codes as A and up
// to 8 NT columns of activations (a row of x, or one of its two planes) as B.
// A 4-bit code in the low bits of a float16 word is the subnormal c 2^-24
// (c 2^-20 four bits higher): one AND makes an operand of two codes.  With one
// plane the zero is taken off after the group's sum, s (sum(c x) - z sum(x));
// with two (fp32), where the sum's last bits count, code and zero become the
// normal number (c - z) 2^-10 by one fma.  The warps' sums are added in order
// through shared memory.
//
// Measured: 8 experts' gate/up (28672 x 4096 each, 16 products, bf16) 88 us, 499
// MB at 5.7 TB/s, 82 instructions a record; their down products (4096 x 14336,
// fp32) 50 us in two parts (both products and the sum back to back: 140 us, 142
// with one part, 3.46 turns of the blocks).  16 rows of 32000 x 2048 (bf16) 22.6
// us with their operands' kernel: 4 records a warp between two joins, 16 warps an
// SM, waiting for records most of the time; one row of 2048 x 2048 (fp32) 6.2 us
// with its launch.  The launch bounds are what groups of 128 need; with groups of
// 64 and 32, whose params take two and four times the registers, some variants
// spill (up to 412 bytes).
//
// kInline: few activations (product() below) are made operands by every block
// for itself, in shared memory, instead of by a kernel of their own; that saves
// a launch where launches are what a product costs.
template <class T, int MT, int NT, int kPer, bool kInline>
__global__ void __launch_bounds__(w4_threads(NT), w4_blocks(MT, NT)) w4_matvec_kernel(MatvecArgs a, PlanesArgs xa) {
    static_assert(!kInline || NT == 1, "inline operands have one column tile");
    constexpr int kPlanes = sizeof(T) == 4 ? 2 : 1;
    constexpr int kThreads = w4_threads(NT), kWarps = kThreads / 32;
    constexpr int kTokens = 8 * NT / kPlanes;                    // products per pass
    constexpr int kV = kPlanes == 2 ? 2 : 4;                     // sums per lane, tile and column tile
    constexpr int kDepth = NT == 2 ? 2 : 4 / MT, kUnroll = kDepth < 2 ? 2 : kDepth;
    constexpr int kRecord = w4_record(kPer), kStep = 4 * kRecord * kWarps;   // from a warp's block of columns to its next
    constexpr uint32_t kEven = 0x000f000fu, kOdd = 0x00f000f0u;
    __shared__ float part[kWarps][MT * 16][kTokens + 1];
    __shared__ Sorted sorted;
    __shared__ float units[8];
    __shared__ int largest[8];
    __shared__ bool infinite;           // a row of x that the block has seen holds an infinity
    extern __shared__ __align__(16) uint4 inline_x[];   // [block * 4 + w][column][4 j], then the sums
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, j = lane & 3;
    if (threadIdx.x == 0) infinite = false;
    sort_products<kThreads, kPlanes>(sorted, a.matrix, a.num_rows, a.E);
    const int items = sorted.used * a.groups.d;

    uint4 code[kDepth][MT][2];
    uint32_t par[kDepth][MT][2 * kPer];
    const uint8_t* base = nullptr;     // the item's records, at the lane's place
    // The item's matrix, tile and part of the columns: blocks [kb_first, kb_last).
    struct Place {
        int m, tile, part;
    };
    auto place_of = [&](int item) {
        Place p;
        p.m = a.groups.div(item);
        const int i = item - p.m * a.groups.d;
        p.part = i >= a.groups_part;
        p.tile = (i - p.part * a.groups_part) * MT;
        return p;
    };
    int kb_first = 0, kb_last = 0;
    auto begin = [&](int item) {
        const Place p = place_of(item);
        kb_first = p.part * a.blocks_part + warp;
        kb_last = min(a.blocks, (p.part + 1) * a.blocks_part);
        base = a.records + ((long long)sorted.matrix[p.m] * (a.tiles / 4) + p.tile / 4) * a.blocks * (4 * kRecord) +
               (p.tile % 4) * kRecord + kb_first * (4 * kRecord);
    };
    // Records of the warp's d-th block of columns from `at` on; the ring's place d.
    const uint32_t code_at = lane * 16, par_at = 1024 + g * (8 * kPer);
    auto fetch = [&](const uint8_t* at, int d, int t, bool live) {
        if (live) {
            const uint8_t* rec = at + t * kRecord;
            code[d][t][0] = load_stream(reinterpret_cast<const uint4*>(rec + code_at));
            code[d][t][1] = load_stream(reinterpret_cast<const uint4*>(rec + code_at + 512));
            const uint8_t* p = rec + par_at;
            if constexpr (kPer == 1) {
                const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
                par[d][t][0] = v.x, par[d][t][1] = v.y;
            } else {
#pragma unroll
                for (int i = 0; i < 2 * kPer; i += 4) {
                    const uint4 v = __ldg(reinterpret_cast<const uint4*>(p) + i / 4);
                    par[d][t][i] = v.x, par[d][t][i + 1] = v.y, par[d][t][i + 2] = v.z, par[d][t][i + 3] = v.w;
                }
            }
        }
    };
    auto fetch_first = [&]() {
#pragma unroll
        for (int d = 0; d < kDepth; ++d)
#pragma unroll
            for (int t = 0; t < MT; ++t) fetch(base + d * kStep, d, t, kb_first + d * kWarps < kb_last);
    };
    int item = blockIdx.x, t0 = 0;
    if (item < items) {
        begin(item);
        fetch_first();
    }
    wait_predecessor_grid();
    launch_dependents();
    if (a.matrix) {   // zeros for the products without a matrix
        for (int i = blockIdx.x * kWarps + warp; i < a.num_rows; i += gridDim.x * kWarps)
            if (sorted.of[i] < 0)
                for (int r = lane; r < a.outputs; r += 32) store_as(a.y, (long long)i * a.outputs + r, 0.0f, a.dtype);
    }

    // The operands of `tokens` products from `rows` on, at most 8 columns.
    int made_m = -1, made_t0 = -1, made_row = -1;
    auto make_x = [&](const short* rows, int tokens) {
        const int columns = tokens * kPlanes, chunks = a.blocks * (kBlockK / 8);
        constexpr int kChunks = kBlockK / kPer / 8;      // of a group
        float* sums = reinterpret_cast<float*>(inline_x + a.blocks * 16 * columns);
        __syncthreads();
        if (threadIdx.x < tokens) largest[threadIdx.x] = 0;
        __syncthreads();
        auto row_of = [&](int t) { return static_cast<const T*>(xa.x) + a.x_share.div(rows[t]) * xa.stride; };
        for (int t = 0; t < tokens; ++t) {
            const T* p = row_of(t);
            float mx = 0.0f;
            for (int c = threadIdx.x; c < chunks; c += kThreads) {
                float v[8];
                load_chunk(p, c * 8, xa.cols, xa.vec, v);
                mx = fmaxf(mx, chunk_max(v));
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            if (lane == 0) atomicMax(largest + t, __float_as_int(mx));   // not negative: ordered as integers
        }
        __syncthreads();
        for (int t = 0; t < tokens; ++t) {
            const T* p = row_of(t);
            const RowScale scale(__int_as_float(largest[t]));
            if (threadIdx.x == 0) units[t] = scale.unit;
            for (int c = threadIdx.x; c < chunks; c += kThreads) {       // whole groups of lanes
                float v[8], sum = 0.0f;
                load_chunk(p, c * 8, xa.cols, xa.vec, v);
#pragma unroll
                for (int i = 0; i < 8; ++i) sum += v[i] *= scale.up;
                uint4 b[kPlanes];
                operands<kPlanes>(v, b);
#pragma unroll
                for (int k = 0; k < kPlanes; ++k) inline_x[(c / 4 * columns + t * kPlanes + k) * 4 + c % 4] = b[k];
                if constexpr (kPlanes == 1) {
                    const unsigned live = chunk_lanes(c, chunks);
#pragma unroll
                    for (int o = 1; o < kChunks; o <<= 1) sum += __shfl_xor_sync(live, sum, o);
                    if (c % kChunks == 0) sums[c / kChunks * 8 + t] = sum * (1.0f / 1048576.0f);
                }
            }
        }
        __syncthreads();
    };

    while (item < items) {
        const auto [m, tile, part_of] = place_of(item);
        const short* rows = sorted.rows + sorted.first[m];
        const int n = sorted.first[m + 1] - sorted.first[m];
        // The lane's part of B, and the sums of the columns whose products it
        // holds; columns past the last product are not read, nor their sums.
        const int columns = min(kTokens, n - t0) * kPlanes;
        const uint4* bx;
        const float* sx;
        int x_block, x_word, x_step = 0, s_step = 0;   // from block to block, word to word, column tile to column tile
        if constexpr (kInline) {
            const int row = a.x_share.div(rows[t0]);
            // One product's row may serve several matrices.
            if (!(made_m == m && made_t0 == t0) && !(columns == kPlanes && made_row == row)) make_x(rows + t0, columns / kPlanes);
            made_m = m, made_t0 = t0, made_row = columns == kPlanes ? row : -1;
            bx = inline_x + lane;
            sx = reinterpret_cast<const float*>(inline_x + a.blocks * 16 * columns) + 2 * j;
            x_word = columns * 4;
            x_block = 4 * x_word;
        } else {
            const long long x_tile = sorted.tile[m] + t0 * kPlanes / 8;
            bx = a.x.plane + x_tile * a.blocks * 128 + lane;
            sx = a.x.sums + x_tile * a.blocks * (kPer * 8) + 2 * j;
            x_block = 128, x_word = 32;
            x_step = a.blocks * 128, s_step = a.blocks * (kPer * 8);
        }
        const int live = (n - t0) * kPlanes - g;      // of the lane's columns c * 8 + g those below
        uint4 bw[2][NT][4];
        auto fetch_x = [&](uint4 (&b)[NT][4], int kb) {
            if (kb < kb_last) {
#pragma unroll
                for (int c = 0; c < NT; ++c)
                    if (c * 8 < live) {
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            const uint4* from = bx + c * x_step + kb * x_block + w * x_word;
                            if constexpr (kInline) b[c][w] = *from;
                            else b[c][w] = __ldg(from);
                        }
                    }
            }
        };
        fetch_x(bw[0], kb_first);
        fetch_x(bw[1], kb_first + kWarps);

        float y[MT][NT][kV];
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int c = 0; c < NT; ++c)
#pragma unroll
                for (int i = 0; i < kV; ++i) y[t][c][i] = 0.0f;

        for (int kb0 = kb_first; kb0 < kb_last; kb0 += kUnroll * kWarps) {
#pragma unroll
            for (int d = 0; d < kUnroll; ++d) {
                const int kb = kb0 + d * kWarps, slot = d % kDepth;
                if (kb >= kb_last) break;
                const bool more = kb + kDepth * kWarps < kb_last;
                float sums[NT][2][kPer];
                if constexpr (kPlanes == 1) {
#pragma unroll
                    for (int c = 0; c < NT; ++c)
#pragma unroll
                        for (int q = 0; q < kPer; ++q) {
                            const float2* from = reinterpret_cast<const float2*>(sx + c * s_step + (kb * kPer + q) * 8);
                            float2 v;
                            if constexpr (kInline) v = *from;
                            else v = __ldg(from);
                            sums[c][0][q] = v.x, sums[c][1][q] = v.y;
                        }
                }
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    const uint4 c0 = code[slot][t][0], c1 = code[slot][t][1];
                    const uint32_t lo[4] = {c0.x, c0.y, c0.z, c0.w}, hi[4] = {c1.x, c1.y, c1.z, c1.w};
#pragma unroll
                    for (int q = 0; q < kPer; ++q) {
                        float acc[NT][4];
                        __half2 zero[2];
                        if constexpr (kPlanes == 2) {
#pragma unroll
                            for (int h = 0; h < 2; ++h)
                                zero[h] = __hmul2(__high2half2(*reinterpret_cast<const __half2*>(&par[slot][t][h * kPer + q])),
                                                  __float2half2_rn(-1.0f / 1024.0f));
                        }
                        auto operand = [&](uint32_t word, uint32_t mask, int h) -> uint32_t {
                            uint32_t v = word & mask;
                            if constexpr (kPlanes == 2) {
                                const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&v),
                                                          __float2half2_rn(mask == kEven ? 16384.0f : 1024.0f), zero[h]);
                                v = *reinterpret_cast<const uint32_t*>(&r);
                            }
                            return v;
                        };
#pragma unroll
                        for (int w = q * (4 / kPer); w < (q + 1) * (4 / kPer); ++w)
#pragma unroll
                            for (int half = 0; half < 2; ++half) {
                                const uint32_t l = lo[w] >> (8 * half), u = hi[w] >> (8 * half);
                                const uint32_t f[4] = {operand(l, kEven, 0), operand(u, kEven, 1),
                                                       operand(l, kOdd, 0), operand(u, kOdd, 1)};
#pragma unroll
                                for (int c = 0; c < NT; ++c) {
                                    const uint4 b = bw[d % 2][c][w];
                                    const uint32_t b0 = half ? b.z : b.x, b1 = half ? b.w : b.y;
                                    if (w == q * (4 / kPer) && half == 0) mma_f16_first(acc[c], f, b0, b1);
                                    else mma_f16(acc[c], f, b0, b1);
                                }
                            }
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&par[slot][t][h * kPer + q]));
#pragma unroll
                            for (int c = 0; c < NT; ++c) {
                                if constexpr (kPlanes == 2) {
                                    y[t][c][h] = fmaf(p.x, fmaf(acc[c][2 * h + 1], 1.0f / 2048.0f, acc[c][2 * h]), y[t][c][h]);
                                } else {
#pragma unroll
                                    for (int i = 0; i < 2; ++i) {
                                        const float v = fmaf(-p.y, sums[c][i][q], acc[c][2 * h + i]);
                                        y[t][c][2 * h + i] = fmaf(p.x, v, y[t][c][2 * h + i]);
                                    }
                                }
                            }
                        }
                    }
                    fetch(base + kDepth * kStep, slot, t, more);
                }
                base += kStep;
                fetch_x(bw[d % 2], kb + 2 * kWarps);
            }
        }
        int next = item, next_t0 = t0 + kTokens;
        if (next_t0 >= n) {
            next = item + gridDim.x;
            next_t0 = 0;
        }
        if (next < items) {
            begin(next);
            fetch_first();
        }
        __syncthreads();   // the last item's sums are read
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int c = 0; c < NT; ++c)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if constexpr (kPlanes == 2) {
                        part[warp][t * 16 + 8 * h + g][c * 4 + j] = y[t][c][h];
                    } else {
                        part[warp][t * 16 + 8 * h + g][c * 8 + 2 * j] = y[t][c][2 * h];
                        part[warp][t * 16 + 8 * h + g][c * 8 + 2 * j + 1] = y[t][c][2 * h + 1];
                    }
                }
        __syncthreads();
        const int now = min(kTokens, n - t0);
        const int out_rows = a.gated ? MT * 8 : MT * 16;
        for (int i = threadIdx.x; i < out_rows * now; i += kThreads) {
            const int r = i % out_rows, token = i / out_rows;
            const int product = rows[t0 + token];
            const float unit = kInline ? units[token] : __ldg(a.x.unit + a.x_share.div(product));
            if (isinf(unit)) infinite = true;
            auto total = [&](int row) {
                float v = 0.0f;
#pragma unroll
                for (int k = 0; k < kWarps; ++k) v += part[k][row][token];
                return v * (kPlanes == 2 ? 1024.0f : 1048576.0f) * unit;   // unit times the power may pass 2^127
            };
            float v;
            int out;
            if (a.gated) {
                const int pair = r / 16;
                v = total(pair * 32 + r % 16);
                v = v / (1.0f + expf(-v)) * total(pair * 32 + 16 + r % 16);
                out = (tile / 2 + pair) * 16 + r % 16;
            } else {
                v = total(r);
                out = tile * 16 + r;
            }
            if (out < a.outputs) store_as(a.y, ((long long)part_of * a.num_rows + product) * a.outputs + out, v, a.dtype);
        }
        item = next;
        t0 = next_t0;
    }

    // The products of rows that hold an infinity once more, in place of what the
    // operands gave for them.
    __syncthreads();
    if (!infinite) return;
    const int x_bytes = xa.dtype == MOE_DTYPE_F32 ? 4 : 2, out_rows = a.gated ? MT * 8 : MT * 16;
    for (item = blockIdx.x; item < items; item += gridDim.x) {
        const Place at = place_of(item);
        const short* rows = sorted.rows + sorted.first[at.m];
        const int n = sorted.first[at.m + 1] - sorted.first[at.m];
        for (int i = threadIdx.x; i < out_rows * n; i += kThreads) {
            const int r = i % out_rows, product = rows[i / out_rows], x_row = a.x_share.div(product);
            const uint8_t* x = static_cast<const uint8_t*>(xa.x) + x_row * xa.stride * x_bytes;
            if (!(kInline ? has_infinity(x, xa.dtype, xa.cols) : isinf(__ldg(a.x.unit + x_row)))) continue;
            const int t = at.tile + r / 16 * (a.gated ? 2 : 1), out = (a.gated ? t / 2 : t) * 16 + r % 16;
            if (out >= a.outputs) continue;
            const uint8_t* rec = a.records + ((long long)sorted.matrix[at.m] * (a.tiles / 4) + t / 4) * a.blocks * (4 * kRecord) + t % 4 * kRecord;
            const float v = defined_output<kPer>(rec, r % 16, a.gated, at.part * a.blocks_part,
                                                 min(a.blocks, (at.part + 1) * a.blocks_part), x, xa.dtype, xa.cols);
            store_as(a.y, ((long long)at.part * a.num_rows + product) * a.outputs + out, v, a.dtype);
        }
    }
}

// y[t] = sum over s of w[t][s] * part[t * k + s], s ascending; with `second`
// not 0 a product's second part lies that many values on.
template <class T>
__global__ void __launch_bounds__(256) experts_sum_kernel(const float* part, const int* idx, const float* w, T* y, int k, int d,
                                                         int E, long long second) {
    const int n = blockIdx.x * 256 + threadIdx.x, t = blockIdx.y;
    wait_predecessor_grid();
    if (n >= d) return;
    float v = 0.0f;
    for (int s = 0; s < k; ++s) {
        const int e = idx[t * k + s];
        if (e < 0 || e >= E) continue;
        const float* p = part + ((long long)t * k + s) * d + n;
        v = fmaf(w[t * k + s], second ? p[0] + p[second] : p[0], v);
    }
    y[(long long)t * d + n] = from_f32<T>(v);
}

}  // namespace
}  // namespace moe

using namespace moe;

struct MoeW4 {
    MoeW4Config cfg;
    int outputs = 0, tiles = 0, blocks = 0, sms = 0;
    uint8_t* records = nullptr;   // with the first workspaces behind them
    Planes x{};               // the activations' operand, of work_rows rows
    float* result = nullptr;  // fp32 results of the experts, result_size values
    size_t result_size = 0;
    int work_rows = 0;
    std::vector<void*> held;  // further workspaces, outgrown ones too: enqueued work and graphs name them
    size_t bytes = 0;
};

namespace {

// A further workspace.  Nothing is freed before the handle is, and nothing
// waited for: what is enqueued or was captured with a smaller one keeps it.
int hold(MoeW4* h, size_t bytes, cudaStream_t s, uint8_t** out) {
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(s, &capture) != cudaSuccess) cudaGetLastError();
    else if (capture != cudaStreamCaptureStatusNone)
        return report_error(MOE_ERR_UNSUPPORTED, "4-bit weights: this call needs more workspace than the handle has, which a "
                                                 "stream capture does not allow; create it with a larger max_rows, or make a "
                                                 "call of this size before the capture");
    h->held.reserve(h->held.size() + 1);
    void* p = nullptr;
    const cudaError_t e = handle_alloc(h->cfg.device, bytes, &p);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return e == cudaErrorMemoryAllocation ? report_error(MOE_ERR_OOM, "4-bit weights: workspace allocation failed")
                                              : launch_status(e, "4-bit weights: workspace allocation");
    }
    h->held.push_back(p);
    h->bytes += bytes;
    *out = static_cast<uint8_t*>(p);
    return MOE_OK;
}

// Bytes of the operands of `rows` products: planes, sums, units.  Column tiles:
// two columns a product, one not full for each matrix in use, and one that the
// last pass of a kernel of two column tiles may look at.
struct OperandBytes {
    size_t plane, sums, unit;
    OperandBytes(const MoeW4* h, int rows) {
        const size_t tiles = rows ? (size_t)(2 * rows + 7) / 8 + std::min(rows, h->cfg.num_matrices) + 1 : 0;
        plane = tiles * h->blocks * 2048;
        sums = tiles * h->blocks * (kBlockK / h->cfg.group) * 8 * sizeof(float);
        unit = ((size_t)rows * sizeof(float) + 255) / 256 * 256;
    }
    size_t all() const { return plane + sums + unit; }
};

void place_operands(MoeW4* h, int rows, uint8_t* at) {
    const OperandBytes b(h, rows);
    h->x = Planes{reinterpret_cast<uint4*>(at), reinterpret_cast<float*>(at + b.plane), reinterpret_cast<float*>(at + b.plane + b.sums)};
    h->work_rows = rows;
}

// A handle that outgrows its operands at least doubles them, so that what it
// holds stays below twice the last.
int ensure_rows(MoeW4* h, int rows, cudaStream_t s) {
    if (rows <= h->work_rows) return MOE_OK;
    rows = std::max(rows, std::min(2 * h->work_rows, kMaxRows));
    uint8_t* at = nullptr;
    const int rc = hold(h, OperandBytes(h, rows).all(), s, &at);
    if (rc == MOE_OK) place_operands(h, rows, at);
    return rc;
}

// Lets the kernels that make operands for themselves have kInlineMax bytes.
template <class T, int kPer> cudaError_t inline_attributes() {
    cudaError_t e = cudaFuncSetAttribute(w4_matvec_kernel<T, 1, 1, kPer, true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         kInlineMax);
    if (e == cudaSuccess)
        e = cudaFuncSetAttribute(w4_matvec_kernel<T, 2, 1, kPer, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kInlineMax);
    return e;
}
template <int kPer> cudaError_t inline_attributes_all() {
    cudaError_t e = inline_attributes<float, kPer>();
    if (e == cudaSuccess) e = inline_attributes<__nv_bfloat16, kPer>();
    if (e == cudaSuccess) e = inline_attributes<__half, kPer>();
    return e;
}

// Room for the experts' fp32 results of a product: two parts where it may be
// split (launch_product), which is the down product.
size_t result_row(const MoeW4* h) { return (size_t)h->outputs * (h->cfg.gated ? 1 : 2); }

int ensure_result(MoeW4* h, int rows, cudaStream_t s) {
    const size_t row = result_row(h);
    if (rows * row <= h->result_size) return MOE_OK;
    const size_t n = std::max(rows * row, std::min(2 * h->result_size, kMaxRows * row));
    uint8_t* at = nullptr;
    const int rc = hold(h, n * sizeof(float), s, &at);
    if (rc != MOE_OK) return rc;
    h->result = reinterpret_cast<float*>(at);
    h->result_size = n;
    return MOE_OK;
}

int w4_create(const MoeW4Config* cfg, const uint8_t* codes, const void* scales, const uint8_t* zeros, MoeW4** out,
              bool on_host) {
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
    if (!on_host && (!aligned_to(codes, 4) || !aligned_to(scales, 2)))
        return report_error(MOE_ERR_INVALID, "moe_w4_create: device codes must be 4-byte aligned, scales to their elements");
    OnDevice on(cfg->device);
    int major = 0, sms = 0;
    cudaError_t e = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, cfg->device);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, cfg->device);
    if (e == cudaSuccess)
        e = cfg->group == 128 ? inline_attributes_all<1>() : cfg->group == 64 ? inline_attributes_all<2>() : inline_attributes_all<4>();
    if (e != cudaSuccess) return launch_status(e, "moe_w4_create");
    if (!on.ok) return report_error(MOE_ERR_CUDA, "moe_w4_create: cannot select the device");
    if (major != 10) return report_error(MOE_ERR_UNSUPPORTED, "libmoe_b200 is built for sm_100a (B200) only");
    std::unique_ptr<MoeW4, void (*)(MoeW4*)> owner(new MoeW4, moe_w4_destroy);
    MoeW4* h = owner.get();
    h->cfg = *cfg;
    h->sms = sms;
    h->outputs = cfg->gated ? cfg->rows / 2 : cfg->rows;
    // Whole quads of tiles, so that a block of any tile count stays inside.
    h->tiles = ((h->outputs + 15) / 16 * (cfg->gated ? 2 : 1) + 3) / 4 * 4;
    h->blocks = (cfg->cols + kBlockK - 1) / kBlockK;
    const int per = kBlockK / cfg->group, groups = (cfg->cols + cfg->group - 1) / cfg->group;
    const size_t matrix = (size_t)h->tiles * h->blocks * w4_record(per), E = cfg->num_matrices;
    // One block for the records, the operands and the experts' results; a matrix that is neither
    // gated nor one of several is not asked for those.
    const size_t records = (matrix * E + 255) / 256 * 256, operands = OperandBytes(h, cfg->max_rows).all();
    if (cfg->gated || cfg->num_matrices > 1) h->result_size = cfg->max_rows * result_row(h);
    h->bytes = records + operands + h->result_size * sizeof(float);
    e = handle_alloc(cfg->device, h->bytes, reinterpret_cast<void**>(&h->records));
    if (e != cudaSuccess) {
        cudaGetLastError();
        return e == cudaErrorMemoryAllocation ? report_error(MOE_ERR_OOM, "moe_w4_create: device allocation failed")
                                              : launch_status(e, "moe_w4_create");
    }
    place_operands(h, cfg->max_rows, h->records + records);
    h->result = reinterpret_cast<float*>(h->records + records + operands);
    // Host weights pass through the device one matrix at a time.
    const size_t nc = (size_t)cfg->rows * (cfg->cols / 2), ng = (size_t)cfg->rows * groups;
    uint8_t* stage = nullptr;
    const size_t scales_at = (nc + 15) / 16 * 16, zeros_at = scales_at + (ng * 2 + 15) / 16 * 16;
    if (on_host) e = cudaMalloc(&stage, zeros_at + ng);
    if (e == cudaSuccess) e = cudaDeviceSynchronize();   // device sources may still be written on any stream
    for (size_t m = 0; m < E && e == cudaSuccess; ++m) {
        PackArgs a{codes + m * nc, static_cast<const __half*>(scales) + m * ng, zeros ? zeros + m * ng : nullptr,
                   h->records + m * matrix, cfg->rows, cfg->cols, cfg->group, h->tiles, h->blocks, cfg->gated != 0};
        if (on_host) {
            e = cudaMemcpy(stage, a.codes, nc, cudaMemcpyHostToDevice);
            if (e == cudaSuccess) e = cudaMemcpy(stage + scales_at, a.scales, ng * 2, cudaMemcpyHostToDevice);
            if (e == cudaSuccess && zeros) e = cudaMemcpy(stage + zeros_at, a.zeros, ng, cudaMemcpyHostToDevice);
            a.codes = stage;
            a.scales = reinterpret_cast<const __half*>(stage + scales_at);
            a.zeros = zeros ? stage + zeros_at : nullptr;
        }
        if (e == cudaSuccess)
            e = launch(w4_pack_kernel, dim3((unsigned)((long long)h->tiles * h->blocks)), 256, 0, nullptr, false, a);
    }
    if (e == cudaSuccess) e = cudaDeviceSynchronize();
    cudaFree(stage);
    const int rc = e == cudaErrorMemoryAllocation ? report_error(MOE_ERR_OOM, "moe_w4_create: device allocation failed")
                                                  : launch_status(e, "moe_w4_create");
    if (rc != MOE_OK) {
        cudaGetLastError();
        return rc;
    }
    *out = owner.release();
    return MOE_OK;
}

// Bytes of `columns` operand columns in shared memory.
size_t inline_bytes(const MoeW4* h, int columns) {
    return (size_t)h->blocks * (columns * 256 + kBlockK / h->cfg.group * 32);
}

template <class T, int MT, int NT, bool kInline>
cudaError_t launch_product(const MoeW4* h, MatvecArgs a, const PlanesArgs& x, int used, int columns, bool dependent,
                           int* parts_out, cudaStream_t s) {
    a.groups_part = (a.tiles_used + MT - 1) / MT;
    // Two parts where they leave the blocks' last turn fuller by a tenth.
    const long long slots = (long long)h->sms * w4_blocks(MT, NT), items = (long long)a.groups_part * used;
    auto filled = [&](long long n) { return (double)n / (double)((n + slots - 1) / slots * slots); };
    constexpr int kWarps = w4_threads(NT) / 32;
    const int parts = parts_out && a.blocks >= 4 * kWarps && filled(2 * items) > filled(items) + 0.1 ? 2 : 1;
    if (parts_out) *parts_out = parts;
    a.blocks_part = (a.blocks + parts * kWarps - 1) / (parts * kWarps) * kWarps;
    a.groups = FastDiv(parts * a.groups_part);
    const dim3 grid((unsigned)std::min(items * parts, slots)), block(w4_threads(NT));
    const size_t smem = kInline ? inline_bytes(h, columns) : 0;
    auto run = [&](auto kernel) { return launch(kernel, grid, block, smem, s, dependent, a, x); };
    switch (kBlockK / h->cfg.group) {
        case 1: return run(w4_matvec_kernel<T, MT, NT, 1, kInline>);
        case 2: return run(w4_matvec_kernel<T, MT, NT, 2, kInline>);
        default: return run(w4_matvec_kernel<T, MT, NT, 4, kInline>);
    }
}

template <class T>
cudaError_t product(const MoeW4* h, const T* x, int num_rows, int64_t x_stride, int x_share, const int* matrix, void* y,
                    int dtype, bool dependent, int* parts, cudaStream_t s) {
    constexpr int kPlanes = sizeof(T) == 4 ? 2 : 1;
    using Plane = std::conditional_t<kPlanes == 2, float, __half>;   // made apart, only the planes count
    const MoeW4Config& c = h->cfg;
    constexpr int x_dtype = kPlanes == 2 ? MOE_DTYPE_F32 : std::is_same_v<T, __half> ? MOE_DTYPE_F16 : MOE_DTYPE_BF16;
    const int x_rows = (num_rows - 1) / x_share + 1;   // num_rows > 0; x_share may be the largest integer
    const PlanesArgs p{x, x_stride, matrix, h->x, c.cols, h->blocks, c.group, num_rows, x_share, matrix ? c.num_matrices : 1,
                       aligned16(x) && x_stride * (int64_t)sizeof(T) % 16 == 0, x_dtype};
    const MatvecArgs a{h->records, h->x, matrix, y, num_rows, matrix ? c.num_matrices : 1, h->tiles, h->blocks, h->outputs, dtype,
                       FastDiv(x_share), FastDiv(), c.gated != 0, (h->outputs + 15) / 16 * (c.gated ? 2 : 1), 0, 0};
    const int used = matrix ? std::min(num_rows, c.num_matrices) : 1;
    const long long work = (long long)a.tiles_used * used;
    // Two tiles of rows a block from 3 of them an SM on (one row bf16, on the GPU: 32000 x 2048 14.4 us
    // against 16.4 with one; 4096 x 8192, 1.7 an SM, 11.2 against 10.3), four from 48 on (experts with 97 an SM
    // 136 us against 140 with two; one row of 65536 x 4096, 28 an SM, 35.8 against 34.6).  Operands are made in every block up to kInlineBlocks (one row bf16
    // 2048 x 2048 6.2 us against 8.2 with a kernel of their own; four rows of 4096 x 4096 12.3 against 8.3).
    const int most = std::min(num_rows * kPlanes, 8);                // columns of a pass
    if (num_rows <= 8 / kPlanes && x_rows * kPlanes * h->blocks <= kInlineBlocks && inline_bytes(h, most) <= kInlineMax &&
        work < 48ll * h->sms)
        return work >= 3ll * h->sms || c.gated ? launch_product<T, 2, 1, true>(h, a, p, used, most, dependent, parts, s)
                                                : launch_product<T, 1, 1, true>(h, a, p, used, most, dependent, parts, s);
    cudaError_t e = launch(w4_planes_kernel<T, kPlanes>, x_rows, 1024, 0, s, dependent, p);
    if (e != cudaSuccess) return e;
    // Columns of a matrix's products: all rows', or twice the mean's where the rows choose their matrices.
    const int columns = kPlanes * (matrix ? std::min(num_rows, 2 * ((num_rows + c.num_matrices - 1) / c.num_matrices)) : num_rows);
    if (columns <= 8)
        return work >= 48ll * h->sms              ? launch_product<Plane, 4, 1, false>(h, a, p, used, 0, true, parts, s)
               : work >= 3ll * h->sms || c.gated ? launch_product<Plane, 2, 1, false>(h, a, p, used, 0, true, parts, s)
                                                  : launch_product<Plane, 1, 1, false>(h, a, p, used, 0, true, parts, s);
    // Two column tiles: one tile of rows leaves registers for a third more warps
    // (16 rows bf16: 32000 x 2048 25.6 us against 27.6 with two, 4096 x 14336 35 against 40).
    return c.gated ? launch_product<Plane, 2, 2, false>(h, a, p, used, 0, true, parts, s)
                   : launch_product<Plane, 1, 2, false>(h, a, p, used, 0, true, parts, s);
}

template <class T>
cudaError_t experts_typed(MoeW4* gu, MoeW4* dn, const void* x, int tokens, int k, const int* idx, const float* w, void* y,
                          cudaStream_t s) {
    int parts = 1;
    cudaError_t e = product(gu, static_cast<const T*>(x), tokens * k, gu->cfg.cols, k, idx, gu->result, MOE_DTYPE_F32,
                            false, nullptr, s);
    if (e == cudaSuccess)
        e = product(dn, gu->result, tokens * k, dn->cfg.cols, 1, idx, dn->result, MOE_DTYPE_F32, true, &parts, s);
    if (e != cudaSuccess) return e;
    return launch(experts_sum_kernel<T>, dim3((dn->outputs + 255) / 256, tokens), 256, 0, s, true, dn->result, idx, w,
                  static_cast<T*>(y), k, dn->outputs, dn->cfg.num_matrices,
                  parts == 2 ? (long long)tokens * k * dn->outputs : 0ll);
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
    return guarded("moe_w4_create", [&] { return w4_create(cfg, codes, scales, zeros, out, true); });
}

int moe_w4_create_from_device(const MoeW4Config* cfg, const uint8_t* codes, const void* scales, const uint8_t* zeros,
                              MoeW4** out) {
    return guarded("moe_w4_create_from_device",
                   [&] { return w4_create(cfg, codes, scales, zeros, out, false); });
}

void moe_w4_destroy(MoeW4* h) {
    if (!h) return;
    OnDevice on(h->cfg.device);
    handle_free(h->records);
    for (void* p : h->held) handle_free(p);
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
        const int rc = ensure_rows(h, num_rows, s);
        if (rc != MOE_OK) return rc;
        cudaError_t e;
        if (dtype == MOE_DTYPE_F32)
            e = product(h, static_cast<const float*>(x), num_rows, x_row_stride, x_share, matrix, y, dtype, false, nullptr, s);
        else if (dtype == MOE_DTYPE_BF16)
            e = product(h, static_cast<const __nv_bfloat16*>(x), num_rows, x_row_stride, x_share, matrix, y, dtype, false, nullptr, s);
        else
            e = product(h, static_cast<const __half*>(x), num_rows, x_row_stride, x_share, matrix, y, dtype, false, nullptr, s);
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
        const cudaStream_t s = static_cast<cudaStream_t>(stream);
        int rc = ensure_rows(gu, T * top_k, s);
        if (rc == MOE_OK) rc = ensure_rows(dn, T * top_k, s);
        if (rc == MOE_OK) rc = ensure_result(gu, T * top_k, s);
        if (rc == MOE_OK) rc = ensure_result(dn, T * top_k, s);
        if (rc != MOE_OK) return rc;
        cudaError_t e = dtype == MOE_DTYPE_F32    ? experts_typed<float>(gu, dn, x, T, top_k, idx, weights, y, s)
                        : dtype == MOE_DTYPE_BF16 ? experts_typed<__nv_bfloat16>(gu, dn, x, T, top_k, idx, weights, y, s)
                                                  : experts_typed<__half>(gu, dn, x, T, top_k, idx, weights, y, s);
        return launch_status(e, "moe_w4_experts_device");
    });
}

}  // extern "C"
