// layer_norm.hip - layer norm over the last dimension and its gradient (include/humanoid_env.h hum_layer_norm*): the
// pre-norm of the policy's memory and the norm of its heads' outputs.  Per row of c channels
//
//     mean = sum x / c,  rstd = 1 / sqrt(sum (x - mean)^2 / c + eps),  h = (x - mean) rstd,  y = w h + b
//     g = w dy,  dx = rstd (g - mean(g) - h mean(g h)),   dw = sum over rows dy h,  db = sum over rows dy
//
// HBM bounds both passes (7 operations an element), so a row is read once into registers and everything else happens
// there: the variance is summed from the differences (two passes over registers, not over memory, and no cancellation).
// TPR threads hold a row, 8 NV channels each, and sum over DPP / LDS.  The backward pass keeps a running dw, db of its
// own channels per thread while its workgroup walks over rows, joins the workgroup's rows in LDS and writes one partial
// row pair per workgroup; a second launch adds those in float64 in a fixed order (no atomics: the same bits each run).
// All sums are float32 or wider; y, dx are rounded once to the rows' type, dw, db once to the weights'.
//
// 131072 x 256 bf16: forward 0.13 GB in 24 us, 5.5 TB/s (a large copy: 5.1); backward 0.20 GB in 44 us a call: 35 (part of
// the rows come from the last cache) and 4 of the second launch, and what lies between launches.  4099 x 1111 float32 at a
// pitch of 1148: backward 15 and 4 us for 55 MB.  One row: 8 us, the host's.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <cstdio>

#include "../../include/humanoid_env.h"
#include "overlap.h"

void hum_internal_set_error(const char* msg);

namespace {

constexpr int MAX_C = 16384;
constexpr int THREADS = 256;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

template <int ST> struct El;
template <> struct El<HUM_F32> { typedef float T; static constexpr int SIZE = 4; };
template <> struct El<HUM_BF16> { typedef __bf16 T; typedef bf16x8 V; static constexpr int SIZE = 2; };
template <> struct El<HUM_F16> { typedef _Float16 T; typedef f16x8 V; static constexpr int SIZE = 2; };

// buffer accesses: a wave's base in scalar registers, a 32-bit byte offset per lane; what lies beyond reads as zero and is
// not written, so a masked lane takes an offset outside instead of a branch (which would make the loads wait for each other)
typedef __amdgpu_buffer_rsrc_t Buf;
constexpr int OUTSIDE = (int)0x80000000;
__device__ __forceinline__ Buf buffer(const void* p, long bytes) {
    return __builtin_amdgcn_make_buffer_rsrc((char*)const_cast<void*>(p) + (p ? bytes : 0), 0, p ? 0x7fffffff : 0, 0x00020000);
}
__device__ __forceinline__ int beyond(int a, int b) { return ~((a - b) >> 31) & OUTSIDE; }   // bit 31 where a >= b

template <int ST>
__device__ __forceinline__ f32x8 load8(Buf b, int at) {
    const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(b, at, 0, 0);
    if constexpr (ST == HUM_F32) {
        const u32x4 w = __builtin_amdgcn_raw_buffer_load_b128(b, at + 16, 0, 0);
        return __builtin_shufflevector(__builtin_bit_cast(f32x4, v), __builtin_bit_cast(f32x4, w), 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
        return __builtin_convertvector(__builtin_bit_cast(typename El<ST>::V, v), f32x8);
    }
}
template <int ST>
__device__ __forceinline__ void store8(Buf b, int at, f32x8 v) {
    if constexpr (ST == HUM_F32) {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, __builtin_shufflevector(v, v, 0, 1, 2, 3)), b, at, 0, 0);
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, __builtin_shufflevector(v, v, 4, 5, 6, 7)), b, at + 16, 0, 0);
    } else {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, __builtin_convertvector(v, typename El<ST>::V)), b, at, 0, 0);
    }
}
template <int ST>
__device__ __forceinline__ float load1(Buf b, int at) {
    if constexpr (ST == HUM_F32) return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(b, at, 0, 0));
    else return (float)__builtin_bit_cast(typename El<ST>::T, (unsigned short)__builtin_amdgcn_raw_buffer_load_b16(b, at, 0, 0));
}
template <int ST>
__device__ __forceinline__ void store1(Buf b, int at, float v) {
    if constexpr (ST == HUM_F32) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, v), b, at, 0, 0);
    else __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, (typename El<ST>::T)v), b, at, 0, 0);
}

// channel of a thread's element i: VEC takes 8 neighbours at a time (16-byte loads), else neighbouring threads take
// neighbouring channels (16-byte loads at any alignment are slower: 49076 x 182 bf16 13.3 us, 16.0; 20000 x 1111 float32 31
// and 37)
template <int TPR, bool VEC>
__device__ __forceinline__ int channel(int j, int i) {
    return VEC ? 8 * ((i / 8) * TPR + j) + i % 8 : i * TPR + j;
}
// a thread's 8 NV channels of a row at byte offset `at` of the buffer (bit 31: no row), zeros behind c
template <int ST, int TPR, int NV, bool VEC>
__device__ __forceinline__ void load_row(Buf b, int at, int j, int c, float (&v)[8 * NV]) {
#pragma unroll
    for (int n = 0; n < NV; n++) {
        if constexpr (VEC) {
            const int e = channel<TPR, true>(j, 8 * n);
            const f32x8 t = load8<ST>(b, (at + e * El<ST>::SIZE) | beyond(e, c));
#pragma unroll
            for (int i = 0; i < 8; i++) v[8 * n + i] = t[i];
        } else {
#pragma unroll
            for (int i = 8 * n; i < 8 * n + 8; i++) {
                const int e = channel<TPR, false>(j, i);
                v[i] = load1<ST>(b, (at + e * El<ST>::SIZE) | beyond(e, c));
            }
        }
    }
}
template <int ST, int TPR, int NV, bool VEC>
__device__ __forceinline__ void store_row(Buf b, int at, int j, int c, const float (&v)[8 * NV]) {
#pragma unroll
    for (int n = 0; n < NV; n++) {
        if constexpr (VEC) {
            const int e = channel<TPR, true>(j, 8 * n);
            f32x8 t;
#pragma unroll
            for (int i = 0; i < 8; i++) t[i] = v[8 * n + i];
            store8<ST>(b, (at + e * El<ST>::SIZE) | beyond(e, c), t);
        } else {
#pragma unroll
            for (int i = 8 * n; i < 8 * n + 8; i++) {
                const int e = channel<TPR, false>(j, i);
                store1<ST>(b, (at + e * El<ST>::SIZE) | beyond(e, c), v[i]);
            }
        }
    }
}
// parameters: float32 or the rows' type
template <int ST, int TPR, int NV, bool VEC>
__device__ __forceinline__ void load_param(const void* p, bool wide, int j, int c, float none, float (&v)[8 * NV]) {
    if (!p) {
#pragma unroll
        for (int i = 0; i < 8 * NV; i++) v[i] = none;
    } else if (wide) {
        load_row<HUM_F32, TPR, NV, VEC>(buffer(p, 0), 0, j, c, v);
    } else {
        load_row<ST, TPR, NV, VEC>(buffer(p, 0), 0, j, c, v);
    }
}
// where the rows of a wave begin: its first row is uniform, a lane's is `below` further (several rows a wave if TPR < 64)
template <int TPR>
struct Place {
    long first;
    int below;
    bool in;
    __device__ __forceinline__ Place(long row0, long rows) {
        constexpr int PER = TPR < 64 ? 64 / TPR : 1;   // rows per wave
        const int t = __builtin_amdgcn_readfirstlane(threadIdx.x & ~63);
        first = row0 + t / TPR;
        below = PER > 1 ? (threadIdx.x & 63) / TPR : 0;
        in = first + below < rows;
    }
    __device__ __forceinline__ int at(long pitch, int size) const { return in ? below * (int)(pitch * size) : OUTSIDE; }
};

// the sum over a row's TPR threads, the same bits in every one of them
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* scratch) {
    constexpr int W = TPR < 64 ? TPR : 64;
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xB1, 0xf, 0xf, false));    // quad [1,0,3,2]
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4E, 0xf, 0xf, false));    // quad [2,3,0,1]
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x141, 0xf, 0xf, false));   // mirror in 8
    if constexpr (W > 8) v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x140, 0xf, 0xf, false));   // mirror in 16
    if constexpr (W > 16) v += __shfl_xor(v, 16);
    if constexpr (W > 32) v += __shfl_xor(v, 32);
    if constexpr (TPR > 64) {
        constexpr int NW = TPR / 64;
        __syncthreads();   // the scratch's last readers are done
        if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int i = 0; i < NW; i++) v += scratch[i];
    }
    return v;
}

struct NormArgs {
    const void* x; const void* w; const void* b; void* y;
    float* mean; float* rstd;
    long rows, x_row, y_row;
    int c, wide;
    float eps;
};

template <int ST, int TPR, int NV, bool VEC>
__global__ void __launch_bounds__(TPR > THREADS ? TPR : THREADS) norm_kernel(NormArgs a) {
    constexpr int N = TPR > THREADS ? TPR : THREADS, GROUPS = N / TPR;
    __shared__ float scratch[N / 64];
    const int j = threadIdx.x % TPR;
    const float inv = 1.f / (float)a.c;
    float w[8 * NV], b[8 * NV];
    load_param<ST, TPR, NV, VEC>(a.w, a.wide, j, a.c, 1.f, w);
    load_param<ST, TPR, NV, VEC>(a.b, a.wide, j, a.c, 0.f, b);
    // every thread of a workgroup makes the same number of turns (row_sum may hold a barrier)
    for (long row0 = (long)blockIdx.x * GROUPS; row0 < a.rows; row0 += (long)gridDim.x * GROUPS) {
        const Place<TPR> row(row0, a.rows);
        float x[8 * NV];
        load_row<ST, TPR, NV, VEC>(buffer(a.x, row.first * a.x_row * El<ST>::SIZE), row.at(a.x_row, El<ST>::SIZE), j, a.c, x);
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 8 * NV; i++) s += x[i];
        const float mean = row_sum<TPR>(s, scratch) * inv;
        s = 0.f;
#pragma unroll
        for (int i = 0; i < 8 * NV; i++) {
            x[i] = channel<TPR, VEC>(j, i) < a.c ? x[i] - mean : 0.f;
            s += x[i] * x[i];
        }
        const float rstd = 1.f / sqrtf(row_sum<TPR>(s, scratch) * inv + a.eps);
#pragma unroll
        for (int i = 0; i < 8 * NV; i++) x[i] = x[i] * rstd * w[i] + b[i];
        store_row<ST, TPR, NV, VEC>(buffer(a.y, row.first * a.y_row * El<ST>::SIZE), row.at(a.y_row, El<ST>::SIZE), j, a.c, x);
        if (j == 0 && a.mean && row.in) {
            a.mean[row.first + row.below] = mean;
            a.rstd[row.first + row.below] = rstd;
        }
    }
}

struct GradArgs {
    const void* dy; const void* x; const void* w; void* dx;
    const float* mean; const float* rstd;
    float* part;   // [workgroup][dw, db][c]; NULL: no parameter gradients
    long rows, dy_row, x_row, dx_row;
    int c, wide;
};

template <int ST, int TPR, int NV, bool VEC>
__global__ void __launch_bounds__(TPR > THREADS ? TPR : THREADS) grad_kernel(GradArgs a) {
    constexpr int N = TPR > THREADS ? TPR : THREADS, GROUPS = N / TPR;
    __shared__ float scratch[N / 64];
    __shared__ float join[2][GROUPS > 1 ? 2 * 8 * NV * TPR : 1];
    const int j = threadIdx.x % TPR, grp = threadIdx.x / TPR;
    const float inv = 1.f / (float)a.c;
    float w[8 * NV], dw[8 * NV], db[8 * NV];
    load_param<ST, TPR, NV, VEC>(a.w, a.wide, j, a.c, 1.f, w);
#pragma unroll
    for (int i = 0; i < 8 * NV; i++) dw[i] = db[i] = 0.f;
    for (long row0 = (long)blockIdx.x * GROUPS; row0 < a.rows; row0 += (long)gridDim.x * GROUPS) {
        const Place<TPR> row(row0, a.rows);
        float x[8 * NV], d[8 * NV];
        load_row<ST, TPR, NV, VEC>(buffer(a.x, row.first * a.x_row * El<ST>::SIZE), row.at(a.x_row, El<ST>::SIZE), j, a.c, x);
        load_row<ST, TPR, NV, VEC>(buffer(a.dy, row.first * a.dy_row * El<ST>::SIZE), row.at(a.dy_row, El<ST>::SIZE), j, a.c, d);
        const float mean = load1<HUM_F32>(buffer(a.mean, row.first * 4), row.at(1, 4)), rstd = load1<HUM_F32>(buffer(a.rstd, row.first * 4), row.at(1, 4));
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < 8 * NV; i++) {
            x[i] = channel<TPR, VEC>(j, i) < a.c ? (x[i] - mean) * rstd : 0.f;
            dw[i] += d[i] * x[i];
            db[i] += d[i];
            d[i] *= w[i];
            s1 += d[i];
            s2 += d[i] * x[i];
        }
        if (a.dx) {
            s1 = row_sum<TPR>(s1, scratch) * inv;
            s2 = row_sum<TPR>(s2, scratch) * inv;
#pragma unroll
            for (int i = 0; i < 8 * NV; i++) d[i] = rstd * (d[i] - s1 - x[i] * s2);
            store_row<ST, TPR, NV, VEC>(buffer(a.dx, row.first * a.dx_row * El<ST>::SIZE), row.at(a.dx_row, El<ST>::SIZE), j, a.c, d);
        }
    }
    if (!a.part) return;
    // the workgroup's rows join: a wave's by exchange, then waves 2 and 3 with 0 and 1, then 1 with 0 (each group of rows over
    // the ones before it through LDS, 62 barriers at 8 threads a row: 1000 x 64 bf16
    // 11.6 us, 6.3 so)
    if constexpr (GROUPS > 1) {
        static_assert(N == 256, "four waves");
#pragma unroll
        for (int step = TPR; step < 64; step *= 2)
#pragma unroll
            for (int i = 0; i < 8 * NV; i++) {
                dw[i] += __shfl_xor(dw[i], step);
                db[i] += __shfl_xor(db[i], step);
            }
        const int wave = threadIdx.x >> 6;
        const bool first = (threadIdx.x & 63) < TPR;
        auto put = [&](float* m) {
            if (first)
#pragma unroll
                for (int i = 0; i < 8 * NV; i++) {
                    m[i * TPR + j] = dw[i];
                    m[(8 * NV + i) * TPR + j] = db[i];
                }
        };
        auto add = [&](const float* m) {
#pragma unroll
            for (int i = 0; i < 8 * NV; i++) {
                dw[i] += m[i * TPR + j];
                db[i] += m[(8 * NV + i) * TPR + j];
            }
        };
        if (wave >= 2) put(join[wave - 2]);
        __syncthreads();
        if (wave < 2) add(join[wave]);
        if (wave == 1) put(join[1]);
        __syncthreads();
        if (wave == 0) add(join[1]);
    }
    if (grp == 0) {
        float* p = a.part + (long)blockIdx.x * 2 * a.c;
        if constexpr (VEC) {   // (single words 32 bytes apart: gradient of 200 x 8000 float32 20 us, 12 so)
#pragma unroll
            for (int i = 0; i < 8 * NV; i += 4) {
                const int e = channel<TPR, true>(j, i);
                if (e < a.c) {
                    *(f32x4*)(p + e) = f32x4{dw[i], dw[i + 1], dw[i + 2], dw[i + 3]};
                    *(f32x4*)(p + a.c + e) = f32x4{db[i], db[i + 1], db[i + 2], db[i + 3]};
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8 * NV; i++) {
                const int e = channel<TPR, false>(j, i);
                if (e < a.c) {
                    p[e] = dw[i];
                    p[a.c + e] = db[i];
                }
            }
        }
    }
}

// dw, db from the workgroups' partial rows: 16 columns x 64 strided partial sums per workgroup, joined in order
template <int ST>
__global__ void __launch_bounds__(1024) param_kernel(const float* part, int blocks, int c, void* dw, void* db, int wide) {
    __shared__ double sums[1024];
    const int col = blockIdx.x * 16 + threadIdx.x % 16, k = threadIdx.x / 16;
    double s = 0.;
    if (col < 2 * c) {
#pragma unroll 8
        for (int i = k; i < blocks; i += 64) s += (double)part[(long)i * 2 * c + col];
    }
    sums[threadIdx.x] = s;
    __syncthreads();
    if (k || col >= 2 * c) return;
    s = 0.;
#pragma unroll 8
    for (int i = 0; i < 64; i++) s += sums[i * 16 + threadIdx.x];
    void* o = col < c ? dw : db;
    if (!o) return;
    const int e = col < c ? col : col - c;
    if (wide) ((float*)o)[e] = (float)s;
    else ((typename El<ST>::T*)o)[e] = (typename El<ST>::T)(float)s;
}

int nerr(int code, const char* fn, const char* m) {
    char t[256];
    std::snprintf(t, sizeof t, "%s: %s", fn, m);
    hum_internal_set_error(t);
    return code;
}

struct OnDevice {   // the caller's current device stays what it was
    int old = -1;
    bool ok;
    explicit OnDevice(int d) { ok = hipGetDevice(&old) == hipSuccess && (old == d || hipSetDevice(d) == hipSuccess); }
    ~OnDevice() {
        int now = -1;
        if (old >= 0 && hipGetDevice(&now) == hipSuccess && now != old) (void)hipSetDevice(old);
    }
};

// threads per row: 8 channels a thread as long as a wave holds the row, then more channels, then a whole workgroup
struct Shape { int tpr, nv; };
Shape shape_of(int c, bool near) {   // near: a wave's rows lie within 2^31 bytes
    if (c <= 64 && near) return {8, 1};
    if (c <= 128 && near) return {16, 1};
    if (c <= 256 && near) return {32, 1};
    if (c <= 512) return {64, 1};
    if (c <= 1024) return {64, 2};
    if (c <= 1536) return {64, 3};
    if (c <= 2048) return {256, 1};
    if (c <= 4096) return {256, 2};
    if (c <= 8192) return {1024, 1};
    return {1024, 2};
}
int groups_of(Shape s) { return s.tpr >= THREADS ? 1 : THREADS / s.tpr; }
// workgroups of the backward pass: one per CU at least, up to 4 while their partial rows (16 bytes a channel written and
// read) stay below an eighth of what the rows themselves take (4099 x 1111 float32: 384 workgroups)
long grad_blocks(long rows, Shape s, int size) {
    const long g = groups_of(s), most = (rows + g - 1) / g;
    long want = 3 * rows * size / 128;
    want = want < 256 ? 256 : want > 1024 ? 1024 : want;
    return most < 1 ? 1 : want < most ? want : most;
}

template <int ST, int TPR, int NV>
void launch_norm_v(const NormArgs& a, bool vec, long blocks, hipStream_t s) {
    constexpr int N = TPR > THREADS ? TPR : THREADS;
    if (vec) hipLaunchKernelGGL((norm_kernel<ST, TPR, NV, true>), dim3((unsigned)blocks), dim3(N), 0, s, a);
    else hipLaunchKernelGGL((norm_kernel<ST, TPR, NV, false>), dim3((unsigned)blocks), dim3(N), 0, s, a);
}
template <int ST, int TPR, int NV>
void launch_norm_v(const GradArgs& a, bool vec, long blocks, hipStream_t s) {
    constexpr int N = TPR > THREADS ? TPR : THREADS;
    if (vec) hipLaunchKernelGGL((grad_kernel<ST, TPR, NV, true>), dim3((unsigned)blocks), dim3(N), 0, s, a);
    else hipLaunchKernelGGL((grad_kernel<ST, TPR, NV, false>), dim3((unsigned)blocks), dim3(N), 0, s, a);
}
template <int ST, typename A>
void launch_norm_s(const A& a, Shape sh, bool vec, long blocks, hipStream_t s) {
    if (sh.tpr == 8) launch_norm_v<ST, 8, 1>(a, vec, blocks, s);
    else if (sh.tpr == 16) launch_norm_v<ST, 16, 1>(a, vec, blocks, s);
    else if (sh.tpr == 32) launch_norm_v<ST, 32, 1>(a, vec, blocks, s);
    else if (sh.tpr == 64 && sh.nv == 1) launch_norm_v<ST, 64, 1>(a, vec, blocks, s);
    else if (sh.tpr == 64 && sh.nv == 2) launch_norm_v<ST, 64, 2>(a, vec, blocks, s);
    else if (sh.tpr == 64) launch_norm_v<ST, 64, 3>(a, vec, blocks, s);
    else if (sh.tpr == 256 && sh.nv == 1) launch_norm_v<ST, 256, 1>(a, vec, blocks, s);
    else if (sh.tpr == 256) launch_norm_v<ST, 256, 2>(a, vec, blocks, s);
    else if (sh.nv == 1) launch_norm_v<ST, 1024, 1>(a, vec, blocks, s);
    else launch_norm_v<ST, 1024, 2>(a, vec, blocks, s);
}
template <typename A>
void launch_norm(int type, const A& a, Shape sh, bool vec, long blocks, hipStream_t s) {
    if (type == HUM_BF16) launch_norm_s<HUM_BF16>(a, sh, vec, blocks, s);
    else if (type == HUM_F16) launch_norm_s<HUM_F16>(a, sh, vec, blocks, s);
    else launch_norm_s<HUM_F32>(a, sh, vec, blocks, s);
}

int check_sizes(const char* fn, const hum_norm_args* p) {
    if (!p) return nerr(HUM_ERR_ARG, fn, "null argument");
    if (p->type != HUM_F32 && p->type != HUM_BF16 && p->type != HUM_F16) return nerr(HUM_ERR_ARG, fn, "unknown element type");
    if (p->param_type != HUM_F32 && p->param_type != p->type) return nerr(HUM_ERR_ARG, fn, "parameters must be float32 or of the rows' type");
    if (p->rows < 0 || p->channels < 1 || p->channels > MAX_C) return nerr(HUM_ERR_ARG, fn, "rows must be >= 0 and channels in [1, 16384]");
    const int es = p->type == HUM_F32 ? 4 : 2, ps = p->param_type == HUM_F32 ? 4 : 2;
    if (p->rows && !p->x) return nerr(HUM_ERR_ARG, fn, "x is required");
    if ((uintptr_t)p->x % es || (uintptr_t)p->weight % ps) return nerr(HUM_ERR_ARG, fn, "rows and parameters must be aligned to their elements");
    return HUM_OK;
}
// rows of 8 lanes to a wave at most
bool near(int64_t row, int size) { return row >= 0 && row < (1l << 28) / size; }
bool aligned(const void* p, int64_t row, int size) { return ((uintptr_t)p | (uintptr_t)(row * size)) % 16 == 0; }

// the memory that arguments stand for (overlap.h)
typedef overlap::Bytes Bytes;
Bytes rows_of(const hum_norm_args* p, const void* at, int64_t row, int size) {
    return Bytes(at, (int64_t)p->channels * size).by(p->rows, row * size);
}
Bytes stats_of(const hum_norm_args* p, const float* at) { return Bytes(at, 4 * p->rows); }
Bytes params_of(const hum_norm_args* p, const void* at, int size) { return Bytes(at, (int64_t)p->channels * size); }
// rows that are read, out of the question where `out` replaces them row for row (a row is in registers before it is written)
Bytes rows_read(const hum_norm_args* p, const void* at, int64_t row, int size, const void* out, int64_t out_row) {
    return at == out && (row == out_row || p->rows < 2) ? Bytes() : rows_of(p, at, row, size);
}

int launched(const char* fn) {
    const hipError_t st = hipGetLastError();
    return st == hipSuccess ? HUM_OK : nerr(HUM_ERR_HIP, fn, hipGetErrorString(st));
}

}  // namespace

extern "C" {

int hum_layer_norm(const hum_norm_args* p, const void* bias, float eps, void* y, int64_t y_row, float* mean, float* rstd,
                   void* stream) {
    const char* fn = "hum_layer_norm";
    if (const int rc = check_sizes(fn, p)) return rc;
    const int es = p->type == HUM_F32 ? 4 : 2, ps = p->param_type == HUM_F32 ? 4 : 2;
    if ((p->rows && !y) || (uintptr_t)y % es || (uintptr_t)bias % ps) return nerr(HUM_ERR_ARG, fn, "y is required; rows and parameters must be aligned to their elements");
    if (!mean != !rstd) return nerr(HUM_ERR_ARG, fn, "mean and rstd are wanted together");
    if (((uintptr_t)mean | (uintptr_t)rstd) % 4) return nerr(HUM_ERR_ARG, fn, "mean and rstd must be aligned to 4 bytes");
    if (!(eps >= 0.f) || !std::isfinite(eps)) return nerr(HUM_ERR_ARG, fn, "eps must be finite and >= 0");
    if (!p->rows) return HUM_OK;
    const Bytes writes[] = {rows_of(p, y, y_row, es), stats_of(p, mean), stats_of(p, rstd)};
    const Bytes reads[] = {rows_read(p, p->x, p->x_row, es, y, y_row), params_of(p, p->weight, ps), params_of(p, bias, ps)};
    if (overlap::clash(writes, reads))
        return nerr(HUM_ERR_ARG, fn, "y and the statistics must overlap neither themselves, each other nor an input (y may be x, row for row)");
    const OnDevice dev(p->device);
    if (!dev.ok) return nerr(HUM_ERR_HIP, fn, "hipSetDevice");
    NormArgs a = {p->x, p->weight, bias, y, mean, rstd, (long)p->rows, (long)p->x_row, (long)y_row, p->channels, p->param_type == HUM_F32, eps};
    const Shape sh = shape_of(p->channels, near(p->x_row, es) && near(y_row, es));
    const bool vec = p->channels % 8 == 0 && aligned(p->x, p->x_row, es) && aligned(y, y_row, es) && ((uintptr_t)p->weight | (uintptr_t)bias) % 16 == 0;
    const long g = groups_of(sh), blocks = (p->rows + g - 1) / g;
    launch_norm(p->type, a, sh, vec, blocks < 16384 ? blocks : 16384, (hipStream_t)stream);
    return launched(fn);
}

int hum_layer_norm_workspace(const hum_norm_args* p, uint64_t* bytes) {
    const char* fn = "hum_layer_norm_workspace";
    if (const int rc = check_sizes(fn, p)) return rc;
    if (!bytes) return nerr(HUM_ERR_ARG, fn, "null argument");
    const int es = p->type == HUM_F32 ? 4 : 2;
    const uint64_t a = grad_blocks(p->rows, shape_of(p->channels, true), es), b = grad_blocks(p->rows, shape_of(p->channels, false), es);
    *bytes = (a > b ? a : b) * 2 * p->channels * sizeof(float);
    return HUM_OK;
}

int hum_layer_norm_backward(const hum_norm_args* p, const void* dy, int64_t dy_row, const float* mean, const float* rstd,
                            void* dx, int64_t dx_row, void* d_weight, void* d_bias, void* workspace,
                            uint64_t workspace_bytes, void* stream) {
    const char* fn = "hum_layer_norm_backward";
    if (const int rc = check_sizes(fn, p)) return rc;
    const int es = p->type == HUM_F32 ? 4 : 2, ps = p->param_type == HUM_F32 ? 4 : 2;
    if (p->rows && (!dy || !mean || !rstd)) return nerr(HUM_ERR_ARG, fn, "dy, mean and rstd are required");
    if (((uintptr_t)dy | (uintptr_t)dx) % es || ((uintptr_t)d_weight | (uintptr_t)d_bias) % ps || ((uintptr_t)mean | (uintptr_t)rstd) % 4)
        return nerr(HUM_ERR_ARG, fn, "rows, statistics and parameters must be aligned to their elements");
    const Shape sh = shape_of(p->channels, near(p->x_row, es) && near(dy_row, es) && near(dx_row, es));
    const bool params = d_weight || d_bias;
    uint64_t need = 0;
    if (params)
        if (const int rc = hum_layer_norm_workspace(p, &need)) return rc;
    if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16))
        return nerr(HUM_ERR_ARG, fn, "the workspace is too small (hum_layer_norm_workspace) or not aligned to 16 bytes");
    if (!params && (!p->rows || !dx)) return HUM_OK;
    const Bytes writes[] = {rows_of(p, dx, dx_row, es), Bytes(params ? workspace : nullptr, need)};
    const Bytes reads[] = {rows_read(p, p->x, p->x_row, es, dx, dx_row), rows_read(p, dy, dy_row, es, dx, dx_row),
                           params_of(p, p->weight, ps), stats_of(p, mean), stats_of(p, rstd)};
    // (the second launch writes these: the inputs have been read, the workspace has not)
    const Bytes sums[] = {params_of(p, d_weight, ps), params_of(p, d_bias, ps)};
    if (overlap::clash(writes, reads) || overlap::clash(sums, writes))
        return nerr(HUM_ERR_ARG, fn, "gradients and the workspace must overlap neither themselves, each other nor an input (dx may be x or dy, row for row)");
    const OnDevice dev(p->device);
    if (!dev.ok) return nerr(HUM_ERR_HIP, fn, "hipSetDevice");
    GradArgs a = {dy, p->x, p->weight, dx, mean, rstd, params ? (float*)workspace : nullptr, (long)p->rows, (long)dy_row, (long)p->x_row, (long)dx_row, p->channels, p->param_type == HUM_F32};
    const bool vec = p->channels % 8 == 0 && aligned(p->x, p->x_row, es) && aligned(dy, dy_row, es) && (!dx || aligned(dx, dx_row, es)) && (uintptr_t)p->weight % 16 == 0;
    const long blocks = grad_blocks(p->rows, sh, es);   // no rows: one workgroup writes zero sums
    launch_norm(p->type, a, sh, vec, blocks, (hipStream_t)stream);
    if (params) {
        const dim3 grid((2 * p->channels + 15) / 16);
        if (p->type == HUM_F32) hipLaunchKernelGGL(param_kernel<HUM_F32>, grid, dim3(1024), 0, (hipStream_t)stream, a.part, (int)blocks, p->channels, d_weight, d_bias, a.wide);
        else if (p->type == HUM_BF16) hipLaunchKernelGGL(param_kernel<HUM_BF16>, grid, dim3(1024), 0, (hipStream_t)stream, a.part, (int)blocks, p->channels, d_weight, d_bias, a.wide);
        else hipLaunchKernelGGL(param_kernel<HUM_F16>, grid, dim3(1024), 0, (hipStream_t)stream, a.part, (int)blocks, p->channels, d_weight, d_bias, a.wide);
    }
    return launched(fn);
}

}  // extern "C"
