// decay_attn.hip - linear attention with a decay for each head (include/humanoid_env.h hum_decay_attn*): the memory of
// a recurrent policy beside policy.hip's network.  Per lane and head, with S [dv, dk] in float32:
//
//     S_t = a_t S_{t-1} + v_t k_t^T,   o_t = scale S_t q_t,   a_t = 0 at an episode's first step, else lambda_h
//
// Unrolled, o_t = scale (sum_{s <= t} D[t, s] (q_t . k_s) v_s + lambda^{t+1} S_0 q_t) with D[t, s] = lambda^{t-s} inside
// one episode and 0 across two.  The gradients have the same form with the operands' roles changed:
//
//     dq_t = scale sum_{s <= t} D[t, s] (do_t . v_s) k_s + ...     forwards,  state sum v k^T
//     dk_s = scale sum_{t >= s} D[t, s] (v_s . do_t) q_t + ...     backwards, state sum do q^T
//     dv_s = scale sum_{t >= s} D[t, s] (k_s . q_t) do_t + ...     backwards, the same state transposed
//
// so one kernel, the walk out = walk(x, y, z) with the state sum y z^T, computes all four (struct Role).
//
// The walk goes over chunks of 32 steps.  Inside a chunk it is products of small matrices on the matrix cores:
// P = (Y X^T) masked and weighted by D, O^T = Z^T P + S^T X^T, S = lambda^32 S + (w Y)^T Z.  One wave owns one (lane,
// head, slice of z's channels) and keeps that slice of S in its accumulators for the whole walk; P and S never leave
// registers, because the rows of every A operand are taken in the order
//     matrix row m of tile a  <->  index 8 (m >> 2) + 4 a + (m & 3)   (of 32)
// under which the accumulators of a pair of tiles (lane group g holds rows 4 g .. 4 g + 3 of each) are exactly the 8
// consecutive contraction indexes 8 g .. 8 g + 7 that lane group needs as an operand of the next product.  Only Y^T and
// Z^T (contraction over the steps) go through LDS, read back transposed.
//
// Rounding.  Products of bf16 inputs are exact in the float32 accumulators.  Computed operands are split into bf16
// parts that sum to them: P and the state read by O into two (2^-18 of the value, under the output's own 2^-9), the
// weighted Y that enters the state into three (2^-26, below float32's 2^-24: the state is held in 32 bits).  float32 and
// float16 inputs use the float32 matrix instruction (16 times slower, 153 TFLOP/s on this card) and are not split.
//
// Non-finite values.  A row of Z multiplies zeros of P for the steps that must not see it (earlier steps, other
// episodes), and 0 x inf is NaN: a chunk whose z rows hold one is walked step by step with the unseen rows zeroed, so
// an episode that diverged leaves the next one, and its own earlier steps, untouched.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <cstdio>
#include <type_traits>

#include "../../include/humanoid_env.h"

void hum_internal_set_error(const char* msg);

namespace {

constexpr int CH = 32;             // steps per chunk: the contraction length of one bf16 matrix instruction
constexpr int MAX_D = 128;         // channels per head
constexpr int XCDS = 8;            // consecutive workgroups go to different XCDs
constexpr int NEAR = 8;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

struct Rows {               // [lane, step, head, channel] with unit channel stride
    void* p;
    long lane, step, head;  // strides in elements
    int shared;             // heads that read one of its heads
    int vec;                // 8 channels are 16 aligned bytes, steps do not overlap, 32 of them span less than 2^31 bytes
};

struct Role {
    Rows x, y, z, out;
    int dy, dz;             // channels of x, y and of z, out
    int rev;                // walks from the last step to the first
    int out_f32;            // float32 partial results (shared heads' gradients), summed by a second launch
    float s_pair, s_in, s_add;   // the scale's place: on the pairs, on what the entering state gives, on what joins it
    const float* state_in;  // element (y channel i, z channel j) at i sy + j sz; NULL = zeros
    float* state_out;       // NULL = not wanted
    float* through;         // [(lane, head), segment]: what the segment leaves of an entering state; NULL = not wanted
    long sy, sz;            // one of them is 1
    long in_unit, in_seg, out_unit, out_seg;   // from one (lane, head) / segment to the next
    int s_vec;              // the state's rows of unit stride are 16-byte aligned
    int slice0;             // first workgroup part of this role
};

struct WalkArgs {
    Role r[3];
    int nroles, parts;
    int lanes, steps, heads;
    int segs, seg_steps;    // the walk of a (lane, head) is cut into segs pieces of seg_steps (a multiple of 32) steps
    int last_only;          // state_out is the last segment's
    const float* log_decay;
    const unsigned char* reset;
    long reset_lane, reset_step;
    const int* lengths;
};

// ---- buffer accesses: a uniform base in scalar registers, a 32-bit byte offset per lane; loads beyond the buffer's size
// give zeros and stores there do nothing, so a masked lane takes an offset outside instead of a branch (a branch around
// each load made the loads wait for one another: 16 of a 64 x 64 state took 25 800 cycles)
typedef __amdgpu_buffer_rsrc_t Buf;
constexpr int OUTSIDE = (int)0x80000000;
__device__ __forceinline__ Buf buffer(const void* p, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, p ? bytes : 0, 0x00020000);
}
// bit 31 where a is not below b: or'ed into an offset it puts it outside (no compare and select, no branch)
__device__ __forceinline__ int beyond(int a, int b) { return ~((a - b) >> 31) & OUTSIDE; }
__device__ __forceinline__ u32x4 buf_load(Buf b, int off) { return __builtin_amdgcn_raw_buffer_load_b128(b, off, 0, 0); }
__device__ __forceinline__ void buf_store(Buf b, int off, u32x4 v) { __builtin_amdgcn_raw_buffer_store_b128(v, b, off, 0, 0); }
__device__ __forceinline__ f32x4 buf_load4(Buf b, int off) { return __builtin_bit_cast(f32x4, buf_load(b, off)); }
__device__ __forceinline__ void buf_store4(Buf b, int off, f32x4 v) { buf_store(b, off, __builtin_bit_cast(u32x4, v)); }

// ---- the element types: ST storage, operands of 8 consecutive contraction indexes per lane
template <int ST> struct Num;   // HUM_F32 / HUM_F16: float32 matrix instructions

template <> struct Num<HUM_BF16> {
    typedef bf16x8 Op;
    typedef __bf16 Elem;
    static constexpr int PAD = 8, PARTS = 3, SIZE = 2;
    static __device__ __forceinline__ Op zero() { return Op{}; }
    static __device__ __forceinline__ Op load(Buf b, int off) { return __builtin_bit_cast(Op, buf_load(b, off)); }
    static __device__ __forceinline__ void store(Buf b, int off, f32x8 v) {
        buf_store(b, off, __builtin_bit_cast(u32x4, __builtin_convertvector(v, Op)));   // to nearest, ties to even
    }
    static __device__ __forceinline__ Op load(const void* p, long off, int n) {   // n of 8 elements, any alignment
        const __bf16* e = (const __bf16*)p + off;
        Op v = {};
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (j < n) v[j] = e[j];
        return v;
    }
    static __device__ __forceinline__ void store(void* p, long off, int n, f32x8 v) {
        __bf16* e = (__bf16*)p + off;
        const Op o = __builtin_convertvector(v, Op);
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (j < n) e[j] = o[j];
    }
    static __device__ __forceinline__ bool finite(Op v) {
        const u32x4 u = __builtin_bit_cast(u32x4, v);
        bool bad = false;
#pragma unroll
        for (int i = 0; i < 4; i++) bad |= (u[i] & 0x7f80u) == 0x7f80u || (u[i] & 0x7f800000u) == 0x7f800000u;
        return !bad;
    }
    static __device__ __forceinline__ void mma(f32x4& c, Op a, Op b) {
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    // v as N bf16 parts: each the rounding of what the ones before leave
    template <int N>
    static __device__ __forceinline__ void split(f32x8 v, Op (&o)[N]) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            o[i] = __builtin_convertvector(v, Op);
            if (i + 1 < N) v -= __builtin_convertvector(o[i], f32x8);
        }
    }
    static __device__ __forceinline__ f32x8 wide(Op a) { return __builtin_convertvector(a, f32x8); }
    // rows s0 .. s0 + 7 of column c (4 columns per quarter of 16 lanes: the transposing LDS load)
    static __device__ __forceinline__ void put(Elem* m, Op v) { *(Op*)m = v; }
    static __device__ __forceinline__ Op column(const Elem* m, int pitch, int s0, int c0, int r) {
        typedef __attribute__((address_space(3))) bf16x4 L4;
        const Elem* p = m + (s0 + (r >> 2)) * pitch + c0 + 8 * (r & 3);
        const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((L4*)p);
        const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((L4*)(p + 4 * pitch));
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
};

template <int ST> struct Num {
    typedef f32x8 Op;
    typedef float Elem;
    static constexpr int PAD = 4, PARTS = 1, SIZE = ST == HUM_F16 ? 2 : 4;
    static __device__ __forceinline__ Op zero() { return Op{}; }
    static __device__ __forceinline__ Op load(Buf b, int off) {
        if constexpr (ST == HUM_F16) return __builtin_convertvector(__builtin_bit_cast(f16x8, buf_load(b, off)), Op);
        else return __builtin_shufflevector(buf_load4(b, off), buf_load4(b, off + 16), 0, 1, 2, 3, 4, 5, 6, 7);
    }
    static __device__ __forceinline__ void store(Buf b, int off, f32x8 v) {
        if constexpr (ST == HUM_F16) {
            buf_store(b, off, __builtin_bit_cast(u32x4, __builtin_convertvector(v, f16x8)));
        } else {
            buf_store4(b, off, __builtin_shufflevector(v, v, 0, 1, 2, 3));
            buf_store4(b, off + 16, __builtin_shufflevector(v, v, 4, 5, 6, 7));
        }
    }
    typedef typename std::conditional<ST == HUM_F16, _Float16, float>::type Stored;
    static __device__ __forceinline__ Op load(const void* p, long off, int n) {
        const Stored* e = (const Stored*)p + off;
        Op v = {};
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (j < n) v[j] = (float)e[j];
        return v;
    }
    static __device__ __forceinline__ void store(void* p, long off, int n, f32x8 v) {
        Stored* e = (Stored*)p + off;
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (j < n) e[j] = (Stored)v[j];
    }
    static __device__ __forceinline__ bool finite(Op v) {
        bool bad = false;
#pragma unroll
        for (int i = 0; i < 8; i++) bad |= (__builtin_bit_cast(unsigned, (float)v[i]) & 0x7f800000u) == 0x7f800000u;
        return !bad;
    }
    static __device__ __forceinline__ void mma(f32x4& c, Op a, Op b) {
#pragma unroll
        for (int j = 0; j < 8; j++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    }
    template <int N>
    static __device__ __forceinline__ void split(f32x8 v, Op (&o)[N]) { o[0] = v; }
    static __device__ __forceinline__ f32x8 wide(Op a) { return a; }
    static __device__ __forceinline__ void put(Elem* m, Op v) {
        *(f32x4*)m = __builtin_shufflevector(v, v, 0, 1, 2, 3);
        *(f32x4*)(m + 4) = __builtin_shufflevector(v, v, 4, 5, 6, 7);
    }
    static __device__ __forceinline__ Op column(const Elem* m, int pitch, int s0, int c0, int r) {
        const Elem* p = m + s0 * pitch + c0 + 8 * (r >> 2) + (r & 3);
        Op v;
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = p[j * pitch];
        return v;
    }
};

__device__ __forceinline__ f32x8 pair(f32x4 a, f32x4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }

// LDS operations of one wave execute in order; this keeps the compiler from moving them past each other
__device__ __forceinline__ void lds_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// 4 x 4 transposes inside quads of lanes: v[q] of quad lane i <-> v[i] of quad lane q
__device__ __forceinline__ f32x4 quad_transpose(f32x4 v) {
    const int l = threadIdx.x;
    auto from = [](float x, auto ctrl) {
        return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(ctrl)::value, 0xf, 0xf, false));
    };
    struct X1 { enum { value = 0xB1 }; };   // quad lane ^ 1
    struct X2 { enum { value = 0x4E }; };   // quad lane ^ 2
    const bool odd = l & 1, upper = l & 2;
#pragma unroll
    for (int p = 0; p < 4; p += 2) {
        const float got = from(odd ? v[p] : v[p + 1], X1{});
        if (odd) v[p] = got; else v[p + 1] = got;
    }
#pragma unroll
    for (int p = 0; p < 2; p++) {
        const float got = from(upper ? v[p] : v[p + 2], X2{});
        if (upper) v[p] = got; else v[p + 2] = got;
    }
    return v;
}

// waves per SIMD that the registers are limited for: two hide each other's loads, where the state and operands fit into
// 256 registers
constexpr int walk_waves(int st, int dy, int dz) { return dy * dz * (st == HUM_BF16 ? 1 : 2) <= 4096 ? 2 : 1; }

// One wave per workgroup.  DY, DZ: channels of y and of the z slice rounded up to 32.  FAST: every operand may be accessed
// 16 bytes at a time through buffers; else element by element, at any alignment and stride.
template <int ST, int DY, int DZ, bool FAST>
__global__ void __launch_bounds__(64, walk_waves(ST, DY, DZ)) walk_kernel(WalkArgs a) {
    typedef Num<ST> M;
    typedef typename M::Op Op;
    constexpr int KY = DY / 32, KZ = DZ / 32;
    constexpr int PO = M::PARTS > 1 ? 2 : 1;   // parts of P and of the state's reading
    constexpr int PS = M::PARTS;               // parts of what joins the state
    constexpr int PY = DY + M::PAD, PZ = DZ + M::PAD;
    constexpr bool WEIGH_Y = KY <= KZ;         // the side with fewer tiles carries the weights into the state
    __shared__ __attribute__((aligned(16))) typename M::Elem ly[CH * PY];
    __shared__ __attribute__((aligned(16))) typename M::Elem lz[CH * PZ];
    // lambda^d times the scale's part for d = -31 .. 32 steps, zeros for d < 0: between two steps of a chunk, and from a
    // step to the chunk's end
    __shared__ float pow_pair[2 * CH], pow_add[2 * CH];

    const int l = threadIdx.x, g = l >> 4, r = l & 15;
    // the parts (roles, slices) of one segment read the same rows, and NEAR segments in a row are neighbours in memory (the
    // heads of a lane, lanes of a time-major step): they go to one XCD, one after the other.  Gradient of 4096 lanes x 32
    // steps: 380 us, 407 with NEAR = 1, 377 with 32 (which leaves XCDs idle at few lanes)
    const int block = blockIdx.x, part = block / XCDS % a.parts, turn = block / (XCDS * a.parts);
    const int item = (turn / NEAR * XCDS + block % XCDS) * NEAR + turn % NEAR;
    if (item >= a.lanes * a.heads * a.segs) return;
    const int unit = item / a.segs, seg = item - unit * a.segs;
    const int ri = (a.nroles > 1 && part >= a.r[1].slice0) + (a.nroles > 2 && part >= a.r[2].slice0);
    const Role& R = a.r[ri];
    const int dz0 = (part - R.slice0) * DZ;
    const int b = unit / a.heads, h = unit - b * a.heads;
    const int steps = a.steps;
    int len = steps;
    if (a.lengths) {
        len = __builtin_amdgcn_readfirstlane(a.lengths[b]);
        len = len < 0 ? 0 : len > steps ? steps : len;
    }
    const int rev = R.rev;
    const float lg = a.log_decay[h] * 1.44269504088896340736f;
    auto power = [&](int n) { return n == 0 ? 1.f : __builtin_amdgcn_exp2f(lg * (float)n); };
    pow_pair[l] = l < CH - 1 ? 0.f : R.s_pair * power(l - (CH - 1));
    pow_add[l] = l < CH - 1 ? 0.f : R.s_add * power(l - (CH - 1));
    const int seg0 = seg * a.seg_steps, seg1 = seg + 1 < a.segs ? seg0 + a.seg_steps : steps;
    const int end = len < seg1 ? len : seg1;
    auto row_of = [&](int tile) { return 8 * (r >> 2) + 4 * tile + (r & 3); };

    // ---- rows of a chunk: x by walk step 16 c + r, y and z by step row_of(t)
    auto head_of = [&](const Rows& m) { return (long)b * m.lane + (long)(h / m.shared) * m.head; };
    const long hx = head_of(R.x), hy = head_of(R.y), hz = head_of(R.z), ho = head_of(R.out);
    const unsigned char* marks = a.reset ? a.reset + (long)b * a.reset_lane : nullptr;
    auto time = [&](int n) { return rev ? len - 1 - n : n; };   // of walk step n
    auto steps_from = [&](int n0) { return end - n0 < CH ? end - n0 : CH; };
    // a chunk of L steps as a buffer from its earliest time to its last row's end: the steps behind L lie outside (walking
    // backwards: before it, at negative offsets)
    const int dy = R.dy, dz = R.dz, out_size = R.out_f32 ? 4 : M::SIZE;
    const int sx = (int)R.x.step * M::SIZE, sy = (int)R.y.step * M::SIZE, sz = (int)R.z.step * M::SIZE, so = (int)R.out.step * out_size;
    auto chunk = [&](const void* p, long head, long step, int d, int n0, int L, int size) {
        const char* at = (const char*)p + (head + (long)(rev ? len - n0 - L : n0) * step) * size;
        return buffer(p ? at : nullptr, ((L - 1) * (int)step + d) * size);
    };
    auto row_at = [&](int n, int L, int step) { return (rev ? L - 1 - n : n) * step; };
    Op X[2][KY], Y[2][KY], Z[2][KZ];
    bool mark = false;
    auto load_x = [&](int n0) {
        const int L = steps_from(n0);
        if constexpr (FAST) {
            const Buf bx = chunk(R.x.p, hx, R.x.step, dy, n0, L, M::SIZE);
#pragma unroll
            for (int c = 0; c < 2; c++) {
                const int at = row_at(16 * c + r, L, sx) + 8 * g * M::SIZE;
#pragma unroll
                for (int k = 0; k < KY; k++) X[c][k] = M::load(bx, (at + 32 * k * M::SIZE) | beyond(32 * k + 8 * g, dy));
            }
        } else {
#pragma unroll
            for (int c = 0; c < 2; c++) {
                const int n = 16 * c + r;
                const long at = hx + (long)time(n0 + n) * R.x.step;
#pragma unroll
                for (int k = 0; k < KY; k++) {
                    const int d = 32 * k + 8 * g;
                    X[c][k] = n < L && d < R.dy ? M::load(R.x.p, at + d, R.dy - d) : M::zero();
                }
            }
        }
    };
    auto load_yz = [&](int n0) {
        const int L = steps_from(n0);
        if constexpr (FAST) {
            const Buf by = chunk(R.y.p, hy, R.y.step, dy, n0, L, M::SIZE), bz = chunk(R.z.p, hz, R.z.step, dz, n0, L, M::SIZE);
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const int aty = row_at(row_of(t), L, sy) + 8 * g * M::SIZE, atz = row_at(row_of(t), L, sz) + (dz0 + 8 * g) * M::SIZE;
#pragma unroll
                for (int k = 0; k < KY; k++) Y[t][k] = M::load(by, (aty + 32 * k * M::SIZE) | beyond(32 * k + 8 * g, dy));
#pragma unroll
                for (int k = 0; k < KZ; k++) Z[t][k] = M::load(bz, (atz + 32 * k * M::SIZE) | beyond(dz0 + 32 * k + 8 * g, dz));
            }
        } else {
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const int n = row_of(t);
                const long aty = hy + (long)time(n0 + n) * R.y.step, atz = hz + (long)time(n0 + n) * R.z.step;
#pragma unroll
                for (int k = 0; k < KY; k++) {
                    const int d = 32 * k + 8 * g;
                    Y[t][k] = n < L && d < R.dy ? M::load(R.y.p, aty + d, R.dy - d) : M::zero();
                }
#pragma unroll
                for (int k = 0; k < KZ; k++) {
                    const int d = dz0 + 32 * k + 8 * g;
                    Z[t][k] = n < L && d < R.dz ? M::load(R.z.p, atz + d, R.dz - d) : M::zero();
                }
            }
        }
        // bit j separates the chunk's walk steps j - 1 and j (bit 0 the entering state, bit L the leaving one).  An
        // episode's first step is cut off from what time puts before it, so the backward walk has it one later.
        if (marks) {
            const int n = n0 + l - rev;
            mark = l <= CH && l >= rev && l - rev < CH && n < end && marks[(long)time(n) * a.reset_step] != 0;
        }
    };
    if (seg0 < end) {
        if (R.out.p) load_x(seg0);
        load_yz(seg0);
    }

    // ---- the entering state: tile (i, j) holds y channels 32 (i / 2) + 8 g + 4 (i & 1) + 0..3 of z channel zc(j)
    f32x4 S[2 * KY][2 * KZ];
    auto zc = [&](int j) { return dz0 + 32 * (j >> 1) + 8 * (r >> 2) + 4 * (j & 1) + (r & 3); };
    // rows of unit stride are read 16 bytes at a time: along y directly, along z by one row a quad lane and a transpose
    const bool along_y = R.sy == 1;
    const int quad = along_y ? 0 : r & 3, s_y = along_y ? 1 : dz, s_z = along_y ? dy : 1;
    auto state_at = [&](int i, int j) {   // byte offset of a tile's 16 bytes
        const int y = 32 * (i >> 1) + 8 * g + 4 * (i & 1) + quad, z = zc(j) - quad;
        return 4 * (__mul24(z, s_z) + __mul24(y, s_y)) | beyond(y, dy) | beyond(z, dz);
    };
    {
        const float* s = R.state_in ? R.state_in + (long)unit * R.in_unit + (long)seg * R.in_seg : nullptr;
        if constexpr (FAST) {
            const Buf bs = buffer(s, 4 * dy * dz);
#pragma unroll
            for (int j = 0; j < 2 * KZ; j++)
#pragma unroll
                for (int i = 0; i < 2 * KY; i++) S[i][j] = buf_load4(bs, state_at(i, j));
            if (!along_y)
#pragma unroll
                for (int j = 0; j < 2 * KZ; j++)
#pragma unroll
                    for (int i = 0; i < 2 * KY; i++) S[i][j] = quad_transpose(S[i][j]);
        } else {
#pragma unroll
            for (int j = 0; j < 2 * KZ; j++)
#pragma unroll
                for (int i = 0; i < 2 * KY; i++) {
                    const int y0 = 32 * (i >> 1) + 8 * g + 4 * (i & 1), z = zc(j);
#pragma unroll
                    for (int q = 0; q < 4; q++)
                        S[i][j][q] = s && z < R.dz && y0 + q < R.dy ? s[(long)z * R.sz + (long)(y0 + q) * R.sy] : 0.f;
                }
        }
    }

    float w_in[2];
#pragma unroll
    for (int c = 0; c < 2; c++) w_in[c] = R.s_in * power(16 * c + r + 1 - rev);
    float passed = 1.f;   // what is left of the entering state

    for (int n0 = seg0; n0 < end; n0 += CH) {
        const int L = end - n0 < CH ? end - n0 : CH;
        const bool more = n0 + CH < end;
        // a mark beyond the chunk's last step (its bit L when walking backwards) is this chunk's as well as the first
        // of the next
        const unsigned long long cut = marks ? __ballot(mark) & ((2ull << (L - 1 + rev)) - 1) : 0;
        bool sane = true;
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int k = 0; k < KZ; k++) sane = sane && M::finite(Z[t][k]);
        const bool slow = __any(!sane);

        // the last cut at or before step n of the chunk: step n sees the steps from there on, and what entered the chunk only
        // if there is none
        auto cuts_to = [&](int n) { return cut & ((2ull << n) - 1); };
        auto last_cut = [&](unsigned long long m) { return m ? 63 - __builtin_clzll(m) : 0; };
        int seen[2];
        float wi[2];
#pragma unroll
        for (int c = 0; c < 2; c++) {
            const unsigned long long m = cuts_to(16 * c + r);
            seen[c] = last_cut(m) - 8 * g;
            wi[c] = m ? 0.f : w_in[c];
        }

        lds_order();
#pragma unroll
        for (int t = 0; t < 2; t++) {
#pragma unroll
            for (int k = 0; k < KY; k++) M::put(ly + row_of(t) * PY + 32 * k + 8 * g, Y[t][k]);
#pragma unroll
            for (int k = 0; k < KZ; k++) M::put(lz + row_of(t) * PZ + 32 * k + 8 * g, Z[t][k]);
        }
        lds_order();

        // ---- P^T: rows s, columns t; masked entries are chosen away, not multiplied
        Op P[2][PO];
        if (R.out.p) {
#pragma unroll
            for (int c = 0; c < 2; c++) {
                f32x4 p[2];
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    p[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int k = 0; k < KY; k++) M::mma(p[t], Y[t][k], X[c][k]);
                }
                f32x8 v = pair(p[0], p[1]);
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float w = pow_pair[CH - 1 + 16 * c + r - 8 * g - j];
                    v[j] = w != 0.f && j >= seen[c] ? v[j] * w : 0.f;
                }
                M::template split<PO>(v, P[c]);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        if (more) load_yz(n0 + CH);   // y and z are in LDS: their registers take the next chunk's rows

        // ---- one pass over the chunk's steps, or one per step where a z row is not finite
        for (int lo = 0; lo < L;) {
            const int hi = slow ? lo + 1 : L;
            Op T[2 * KZ];   // Z^T
#pragma unroll
            for (int j = 0; j < 2 * KZ; j++) T[j] = M::column(lz, PZ, 8 * g, 32 * (j >> 1) + 4 * (j & 1), r);
            if (slow) {     // of which step lo sees its episode's, up to itself
                const int from = last_cut(cuts_to(lo));
#pragma unroll
                for (int j = 0; j < 2 * KZ; j++)
#pragma unroll
                    for (int e = 0; e < 8; e++) T[j][e] = 8 * g + e >= from && 8 * g + e < hi ? T[j][e] : (typename M::Elem)0.f;
            }
            // ---- O^T: rows z channels, columns t
            if (R.out.p) {
#pragma unroll
                for (int k = 0; k < KZ; k++) {
                    f32x4 o[2][2];
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const int j = 2 * k + e;
#pragma unroll
                        for (int c = 0; c < 2; c++) o[c][e] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int q = 0; q < KY; q++) {
                            Op sp[PO];
                            M::template split<PO>(pair(S[2 * q][j], S[2 * q + 1][j]), sp);
#pragma unroll
                            for (int u = 0; u < PO; u++)
#pragma unroll
                                for (int c = 0; c < 2; c++) M::mma(o[c][e], sp[u], X[c][q]);
                        }
#pragma unroll
                        for (int c = 0; c < 2; c++) {
#pragma unroll
                            for (int q = 0; q < 4; q++) o[c][e][q] = wi[c] != 0.f ? o[c][e][q] * wi[c] : 0.f;
#pragma unroll
                            for (int u = 0; u < PO; u++) M::mma(o[c][e], T[j], P[c][u]);
                        }
                    }
                    const int d = dz0 + 32 * k + 8 * g;
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        const int n = 16 * c + r;
                        const f32x8 v = pair(o[c][0], o[c][1]);
                        const bool in = n >= lo && n < hi && d < dz;
                        if constexpr (FAST) {
                            const Buf bo = chunk(R.out.p, ho, R.out.step, dz, n0, L, out_size);
                            int at = (row_at(n, L, so) + d * out_size) | beyond(d, dz);
                            if (slow) at = in ? at : OUTSIDE;
                            if (R.out_f32) Num<HUM_F32>::store(bo, at, v);
                            else M::store(bo, at, v);
                        } else if (in) {
                            const long at = ho + (long)time(n0 + n) * R.out.step + d;
                            if (R.out_f32) Num<HUM_F32>::store(R.out.p, at, R.dz - d, v);
                            else M::store(R.out.p, at, R.dz - d, v);
                        }
                    }
                }
                if (hi == L && more) load_x(n0 + CH);
            }
            __builtin_amdgcn_sched_barrier(0);
            // ---- the state behind the chunk
            if (hi == L && (more || R.state_out)) {
                const float through = cut ? 0.f : power(L);
                passed *= through;
                if (!cut) {
#pragma unroll
                    for (int i = 0; i < 2 * KY; i++)
#pragma unroll
                        for (int j = 0; j < 2 * KZ; j++) S[i][j] *= through;
                } else {
#pragma unroll
                    for (int i = 0; i < 2 * KY; i++)
#pragma unroll
                        for (int j = 0; j < 2 * KZ; j++) S[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
                }
                const int leaving = last_cut(cut);
                float wo[8];   // (rows behind the chunk's last step are zeros)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float w = pow_add[CH - 1 + L - 1 + rev - 8 * g - j];
                    wo[j] = 8 * g + j >= leaving ? w : 0.f;
                }
                // nothing joins it where an episode starts right behind (before, in time)
                auto weigh = [&](Op x) {
                    f32x8 v = M::wide(x);
#pragma unroll
                    for (int j = 0; j < 8; j++) v[j] = wo[j] != 0.f ? v[j] * wo[j] : 0.f;
                    return v;
                };
                if (!(cut >> L & 1)) {
                    if constexpr (WEIGH_Y) {
#pragma unroll
                        for (int i = 0; i < 2 * KY; i++) {
                            __builtin_amdgcn_sched_barrier(0);
                            Op yp[PS];
                            M::template split<PS>(weigh(M::column(ly, PY, 8 * g, 32 * (i >> 1) + 4 * (i & 1), r)), yp);
#pragma unroll
                            for (int u = 0; u < PS; u++)
#pragma unroll
                                for (int j = 0; j < 2 * KZ; j++) M::mma(S[i][j], yp[u], T[j]);
                        }
                    } else {
                        Op yt[2 * KY];
#pragma unroll
                        for (int i = 0; i < 2 * KY; i++) yt[i] = M::column(ly, PY, 8 * g, 32 * (i >> 1) + 4 * (i & 1), r);
#pragma unroll
                        for (int j = 0; j < 2 * KZ; j++) {
                            __builtin_amdgcn_sched_barrier(0);
                            Op zp[PS];
                            M::template split<PS>(weigh(T[j]), zp);
#pragma unroll
                            for (int u = 0; u < PS; u++)
#pragma unroll
                                for (int i = 0; i < 2 * KY; i++) M::mma(S[i][j], yt[i], zp[u]);
                        }
                    }
                }
            }
            lo = hi;
        }
    }

    // ---- the steps behind the lane's length
    if (R.out.p)
        for (int n = (len > seg0 ? len : seg0) + r; n < seg1; n += 16)
#pragma unroll
            for (int k = 0; k < KZ; k++) {
                const int d = dz0 + 32 * k + 8 * g;
                if (d < R.dz) {
                    if (R.out_f32) Num<HUM_F32>::store(R.out.p, ho + (long)n * R.out.step + d, R.dz - d, f32x8{});
                    else M::store(R.out.p, ho + (long)n * R.out.step + d, R.dz - d, f32x8{});
                }
            }
    if (R.through && l == 0 && dz0 == 0) R.through[item] = passed;
    if (R.state_out && (!a.last_only || seg + 1 == a.segs)) {
        float* s = R.state_out + (long)unit * R.out_unit + (long)seg * R.out_seg;
        if constexpr (FAST) {
            const Buf bs = buffer(s, 4 * dy * dz);
            if (!along_y)
#pragma unroll
                for (int j = 0; j < 2 * KZ; j++)
#pragma unroll
                    for (int i = 0; i < 2 * KY; i++) S[i][j] = quad_transpose(S[i][j]);
#pragma unroll
            for (int j = 0; j < 2 * KZ; j++)
#pragma unroll
                for (int i = 0; i < 2 * KY; i++) buf_store4(bs, state_at(i, j), S[i][j]);
        } else {
#pragma unroll
            for (int j = 0; j < 2 * KZ; j++)
#pragma unroll
                for (int i = 0; i < 2 * KY; i++) {
                    const int y0 = 32 * (i >> 1) + 8 * g + 4 * (i & 1), z = zc(j);
#pragma unroll
                    for (int q = 0; q < 4; q++)
                        if (z < R.dz && y0 + q < R.dy) s[(long)z * R.sz + (long)(y0 + q) * R.sy] = S[i][j][q];
                }
        }
    }
}

// the segments' entering states from what each of them adds: seg[g] <- state before segment g, one thread per N elements
template <int N>
__global__ void __launch_bounds__(256) scan_kernel(const float* in, float* seg, const float* through, int segs, long units, int size) {
    typedef float V __attribute__((ext_vector_type(N)));
    const long e = ((long)blockIdx.x * 256 + threadIdx.x) * N;
    if (e >= units * size) return;
    const long unit = e / size;
    const int at = (int)(e - unit * size);
    V cur = {};
    if (in) cur = *(const V*)(in + e);
    float* s = seg + unit * segs * size + at;
    const float* th = through + unit * segs;
    constexpr int AHEAD = 8;   // loads in flight
    for (int g0 = 0; g0 < segs; g0 += AHEAD) {
        V add[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; i++)
            if (g0 + i + 1 < segs) add[i] = *(const V*)(s + (long)(g0 + i) * size);
#pragma unroll
        for (int i = 0; i < AHEAD; i++)
            if (g0 + i < segs) {
                *(V*)(s + (long)(g0 + i) * size) = cur;
                if (g0 + i + 1 < segs) {
                    const float t = th[g0 + i];
                    cur = t != 0.f ? cur * t + add[i] : add[i];   // behind a cut nothing of the old state is left
                }
            }
    }
}

// gradients of keys and values that `group` heads share: the sum of the heads' float32 partial results
// part [lanes, steps, heads, d] -> out [lanes, steps, heads / group, d]; one thread per output channel
template <int ST>
__global__ void __launch_bounds__(256) share_kernel(const float* part, Rows out, long rows, int steps, int kv, int group, int d) {
    for (long e = (long)blockIdx.x * 256 + threadIdx.x; e < rows * kv * d; e += (long)gridDim.x * 256) {
        const int c = (int)(e % d);
        const long row = e / d;          // (lane, step, kv head)
        const int g = (int)(row % kv);
        const long bt = row / kv;
        float s = 0.f;
        for (int i = 0; i < group; i++) s += part[((bt * kv + g) * group + i) * d + c];
        const long at = bt / steps * out.lane + bt % steps * out.step + (long)g * out.head + c;
        if constexpr (ST == HUM_F32) ((float*)out.p)[at] = s;
        else if constexpr (ST == HUM_BF16) ((__bf16*)out.p)[at] = (__bf16)s;
        else ((_Float16*)out.p)[at] = (_Float16)s;
    }
}

// ---- single step: S = a S + v k^T, o = scale S q, all in float32 on the vector units - the state is read and written
// once (8 bytes for 4 operations), so HBM bounds it.  LPR lanes of 4 key channels hold one row of S; a wave has
// 64 / LPR rows in one load and U loads in flight, issued before anything that decides whether they are used.
struct StepArgs {
    Rows q, k, v, out;
    const float* log_decay;
    const float* state_in;
    float* state_out;
    const unsigned char* reset;
    long reset_lane;
    const unsigned char* active;
    int heads, dk, dv, blocks;   // blocks: workgroups per (lane, head)
    float scale;
};

template <int ST>
__device__ __forceinline__ float elem(const void* p, long at) {
    if constexpr (ST == HUM_F32) return ((const float*)p)[at];
    else if constexpr (ST == HUM_BF16) return (float)((const __bf16*)p)[at];
    else return (float)((const _Float16*)p)[at];
}

template <int ST>
__device__ __forceinline__ void put_elem(void* p, long at, float v) {
    if constexpr (ST == HUM_F32) ((float*)p)[at] = v;
    else if constexpr (ST == HUM_BF16) ((__bf16*)p)[at] = (__bf16)v;
    else ((_Float16*)p)[at] = (_Float16)v;
}

template <int LPR>
__device__ __forceinline__ float row_sum(float v) {   // over LPR neighbouring lanes, every one of them gets it
    if constexpr (LPR > 1) v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xB1, 0xf, 0xf, false));   // quad [1,0,3,2]
    if constexpr (LPR > 2) v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4E, 0xf, 0xf, false));   // quad [2,3,0,1]
    if constexpr (LPR > 4) v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x141, 0xf, 0xf, false));  // mirror in 8
    if constexpr (LPR > 8) v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x140, 0xf, 0xf, false));  // mirror in 16
    if constexpr (LPR > 16) v += __shfl_xor(v, 16);
    return v;
}

// VEC: rows of S are 16-byte aligned multiples of 4 channels
template <int ST, int LPR, bool VEC>
__global__ void __launch_bounds__(256) step_kernel(StepArgs a) {
    constexpr int U = 4, ROWS = 64 / LPR;
    const int unit = blockIdx.x / a.blocks, blk = blockIdx.x - unit * a.blocks;
    const int b = unit / a.heads, h = unit - b * a.heads;
    const int wave = threadIdx.x >> 6, l = threadIdx.x & 63;
    const int c0 = 4 * (l % LPR), row0 = (blk * 4 + wave) * U * ROWS + l / LPR;
    const long size = (long)a.dv * a.dk;
    const Buf si = buffer(a.state_in ? a.state_in + unit * size : nullptr, 4 * (int)size), so = buffer(a.state_out + unit * size, 4 * (int)size);
    int at[U];   // byte offsets of a lane's 4 channels (VEC), else of the first
    f32x4 s[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int row = row0 + u * ROWS;
        at[u] = 4 * (__mul24(row, a.dk) + c0) | beyond(row, a.dv) | beyond(c0, a.dk);
        if constexpr (VEC) {
            s[u] = buf_load4(si, at[u]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++)
                s[u][j] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(si, (at[u] + 4 * j) | beyond(c0 + j, a.dk), 0, 0));
        }
    }
    const long qo = (long)b * a.q.lane + (long)(h / a.q.shared) * a.q.head, ko = (long)b * a.k.lane + (long)(h / a.k.shared) * a.k.head;
    const long vo = (long)b * a.v.lane + (long)(h / a.v.shared) * a.v.head, oo = (long)b * a.out.lane + (long)h * a.out.head;
    float q[4], k[4], v[U];
#pragma unroll
    for (int j = 0; j < 4; j++) {   // (a channel behind the last reads the last: its k is made 0)
        const int c = c0 + j < a.dk ? c0 + j : a.dk - 1;
        q[j] = elem<ST>(a.q.p, qo + c);
        k[j] = elem<ST>(a.k.p, ko + c);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int row = row0 + u * ROWS;
        v[u] = elem<ST>(a.v.p, vo + (row < a.dv ? row : a.dv - 1));
    }
    const bool on = !a.active || a.active[b];
    const bool fresh = a.reset && a.reset[(long)b * a.reset_lane];
    const float lambda = __builtin_amdgcn_exp2f(a.log_decay[h] * 1.44269504088896340736f);
    const bool keep = !on && a.state_in == a.state_out;   // an idle lane's state in place stays as it is
    float o[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        o[u] = 0.f;
        if (on) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const bool in = c0 + j < a.dk;
                s[u][j] = in ? (fresh ? 0.f : s[u][j] * lambda) + v[u] * k[j] : 0.f;
                o[u] += in ? s[u][j] * q[j] : 0.f;
            }
            o[u] = row_sum<LPR>(o[u]) * a.scale;
        }
        if (!keep) {
            if constexpr (VEC) {
                buf_store4(so, at[u], s[u]);
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++)
                    __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, (float)s[u][j]), so, (at[u] + 4 * j) | beyond(c0 + j, a.dk), 0, 0);
            }
        }
    }
    // every lane of a row has its sum: lane u of the row stores the u-th
    if constexpr (LPR >= U) {
        const int u = l % LPR, row = row0 + u * ROWS;
        const float x = u == 0 ? o[0] : u == 1 ? o[1] : u == 2 ? o[2] : o[3];
        if (u < U && row < a.dv) put_elem<ST>(a.out.p, oo + row, x);
    } else {
#pragma unroll
        for (int u = 0; u < U; u++)
            if (l % LPR == 0 && row0 + u * ROWS < a.dv) put_elem<ST>(a.out.p, oo + row0 + u * ROWS, o[u]);
    }
}

// ------------------------------------------------------------------------------------------------ host side
int derr(int code, const char* fn, const char* m) {
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

int elem_size(int type) { return type == HUM_F32 ? 4 : 2; }

Rows rows_of(const hum_rows& r, int shared, int size, int d) {
    const bool vec = ((uintptr_t)r.ptr | (uintptr_t)(r.lane * size) | (uintptr_t)(r.step * size) | (uintptr_t)(r.head * size)) % 16 == 0 &&
                     d % 8 == 0 && r.step >= d && r.step < (1l << 31) / (CH * size);
    return Rows{r.ptr, (long)r.lane, (long)r.step, (long)r.head, shared, vec};
}

int check_args(const char* fn, const hum_decay_attn_args* p) {
    if (!p) return derr(HUM_ERR_ARG, fn, "null argument");
    if (p->type != HUM_F32 && p->type != HUM_BF16 && p->type != HUM_F16) return derr(HUM_ERR_ARG, fn, "unknown element type");
    if (p->lanes < 0 || p->steps < 0 || p->heads < 1 || p->kv_heads < 1 || p->heads % p->kv_heads)
        return derr(HUM_ERR_ARG, fn, "lanes and steps must be >= 0 and kv_heads must divide heads");
    if (p->dk < 1 || p->dk > MAX_D || p->dv < 1 || p->dv > MAX_D)
        return derr(HUM_ERR_ARG, fn, "dk and dv must be in [1, 128]");
    if ((long)p->lanes * p->heads > (1l << 21)) return derr(HUM_ERR_ARG, fn, "lanes x heads must not pass 2^21");
    if (!std::isfinite(p->scale)) return derr(HUM_ERR_ARG, fn, "scale must be finite");
    if (p->lanes && (!p->log_decay)) return derr(HUM_ERR_ARG, fn, "log_decay is required");
    if (p->lanes && p->steps && (!p->q.ptr || !p->k.ptr || !p->v.ptr)) return derr(HUM_ERR_ARG, fn, "q, k and v are required");
    const hum_rows* all[3] = {&p->q, &p->k, &p->v};
    for (const hum_rows* r : all)
        if (((uintptr_t)r->ptr) % elem_size(p->type)) return derr(HUM_ERR_ARG, fn, "q, k and v must be aligned to their elements");
    if (((uintptr_t)p->state_in | (uintptr_t)p->state_out | (uintptr_t)p->log_decay | (uintptr_t)p->lengths) % 4)
        return derr(HUM_ERR_ARG, fn, "states, log_decay and lengths must be aligned to 4 bytes");
    return HUM_OK;
}

int y_width(int d) { return d <= 32 ? 32 : d <= 64 ? 64 : 128; }
// channels of z per workgroup: 64 for bf16 (P is formed once for them), 32 where float32 matrix instructions take the time
// and twice the waves shorten it (37 lanes x 203 steps, 6 heads, 40 / 72 channels: 51 us, 76 with 64)
int z_slice(int type, int d) { return type != HUM_BF16 || d <= 32 ? 32 : 64; }

template <int ST, int DY, int DZ>
void launch_walk_f(const WalkArgs& a, hipStream_t s) {
    const long units = (long)a.lanes * a.heads * a.segs;
    const dim3 grid((unsigned)((units + XCDS * NEAR - 1) / (XCDS * NEAR) * (XCDS * NEAR) * a.parts));
    bool fast = true;
    for (int i = 0; i < a.nroles; i++) {
        const Role& r = a.r[i];
        fast = fast && (!r.x.p || r.x.vec) && r.y.vec && r.z.vec && (!r.out.p || r.out.vec) && r.s_vec;
    }
    if (fast) hipLaunchKernelGGL((walk_kernel<ST, DY, DZ, true>), grid, dim3(64), 0, s, a);
    else hipLaunchKernelGGL((walk_kernel<ST, DY, DZ, false>), grid, dim3(64), 0, s, a);
}
template <int ST, int DY>
void launch_walk_z(const WalkArgs& a, int dzs, hipStream_t s) {
    if constexpr (ST == HUM_BF16)
        if (dzs == 64) {
            launch_walk_f<ST, DY, 64>(a, s);
            return;
        }
    launch_walk_f<ST, DY, 32>(a, s);
}
template <int ST>
void launch_walk_y(const WalkArgs& a, int dyw, int dzs, hipStream_t s) {
    if (dyw == 32) launch_walk_z<ST, 32>(a, dzs, s);
    else if (dyw == 64) launch_walk_z<ST, 64>(a, dzs, s);
    else launch_walk_z<ST, 128>(a, dzs, s);
}
void launch_walk(int type, const WalkArgs& a, int dyw, int dzs, hipStream_t s) {
    if (type == HUM_BF16) launch_walk_y<HUM_BF16>(a, dyw, dzs, s);
    else if (type == HUM_F16) launch_walk_y<HUM_F16>(a, dyw, dzs, s);
    else launch_walk_y<HUM_F32>(a, dyw, dzs, s);
}

// Few lanes and many steps: the walks are cut into segments that run side by side, each from the state that a first pass
// over the segments before it and a scan have left for it (segments without outputs: half the work of a walk).
struct Cut { int segs, steps; };
constexpr int WAVES = 1024, MIN_CHUNKS = 4;   // one wave per SIMD; segments of 4 chunks at least
Cut cut_of(const hum_decay_attn_args* p, int parts) {
    const long waves = (long)p->lanes * p->heads * parts;
    const int chunks = (p->steps + CH - 1) / CH;
    if (waves == 0 || 2 * waves > WAVES || chunks < 2 * MIN_CHUNKS) return {1, p->steps};
    long segs = WAVES / waves;
    if (segs > chunks / MIN_CHUNKS) segs = chunks / MIN_CHUNKS;
    const int per = (int)((chunks + segs - 1) / segs);
    return {(chunks + per - 1) / per, per * CH};
}

// the roles of equal widths share a launch (their workgroups read the same rows at about the same time)
void launch_roles(const hum_decay_attn_args* p, Role* r, int n, Cut c, bool last_only, hipStream_t s) {
    bool done[3] = {};
    for (int i = 0; i < n; i++) {
        if (done[i]) continue;
        const int dyw = y_width(r[i].dy), dzs = z_slice(p->type, r[i].dz);
        WalkArgs a = {};
        for (int j = i; j < n; j++) {
            if (done[j] || y_width(r[j].dy) != dyw || z_slice(p->type, r[j].dz) != dzs) continue;
            done[j] = true;
            r[j].slice0 = a.parts;
            a.parts += (r[j].dz + dzs - 1) / dzs;
            a.r[a.nroles++] = r[j];
        }
        a.lanes = p->lanes;
        a.steps = p->steps;
        a.heads = p->heads;
        a.segs = c.segs;
        a.seg_steps = c.steps;
        a.last_only = last_only;
        a.log_decay = p->log_decay;
        a.reset = p->reset;
        a.reset_lane = p->reset_lane;
        a.reset_step = p->reset_step;
        a.lengths = p->lengths;
        launch_walk(p->type, a, dyw, dzs, s);
    }
}

// a state [dv, dk] as the walk's sum over (y channel, z channel): y = keys' side or y = values' side
void role_state(Role& r, const float* in, float* out, const hum_decay_attn_args* p, bool y_is_k) {
    r.state_in = in;
    r.state_out = out;
    r.sy = y_is_k ? 1 : p->dk;
    r.sz = y_is_k ? p->dk : 1;
    r.in_unit = r.out_unit = (long)p->dk * p->dv;
    r.s_vec = p->dk % 4 == 0 && ((uintptr_t)in | (uintptr_t)out) % 16 == 0;
}

uint64_t round16(uint64_t n) { return (n + 15) / 16 * 16; }
// scratch of one cut walk: the segments' states, then their `through`
uint64_t walk_bytes(const hum_decay_attn_args* p, Cut c) {
    const uint64_t units = (uint64_t)p->lanes * p->heads * c.segs;
    return c.segs > 1 ? round16(4 * units * p->dk * p->dv) + round16(4 * units) : 0;
}
// fills the scratch with the segments' entering states: `walk` is a role whose y side is the keys' (or queries')
void run_segments(const hum_decay_attn_args* p, Role walk, float* scratch, Cut c, hipStream_t s) {
    const long units = (long)p->lanes * p->heads, size = (long)p->dk * p->dv;
    float* through = (float*)((char*)scratch + round16(4 * units * c.segs * size));
    const float* in = walk.state_in;
    walk.x = Rows{};
    walk.out = Rows{};
    walk.x.shared = walk.out.shared = 1;
    walk.state_in = nullptr;
    walk.state_out = scratch;
    walk.out_unit = size * c.segs;
    walk.out_seg = size;
    walk.through = through;
    walk.s_vec = p->dk % 4 == 0;
    launch_roles(p, &walk, 1, c, false, s);
    if (size % 4 == 0 && (uintptr_t)in % 16 == 0)
        hipLaunchKernelGGL(scan_kernel<4>, dim3((unsigned)((units * size / 4 + 255) / 256)), dim3(256), 0, s, in, scratch, through, c.segs, units, (int)size);
    else
        hipLaunchKernelGGL(scan_kernel<1>, dim3((unsigned)((units * size + 255) / 256)), dim3(256), 0, s, in, scratch, through, c.segs, units, (int)size);
}
void enter_segments(Role& r, const float* scratch, const hum_decay_attn_args* p, Cut c) {
    r.state_in = scratch;
    r.in_unit = (long)p->dk * p->dv * c.segs;
    r.in_seg = (long)p->dk * p->dv;
}
int parts_of(const hum_decay_attn_args* p, int dy, int dz) {
    const int s = z_slice(p->type, dz);
    return (dz + s - 1) / s;
}
Cut forward_cut(const hum_decay_attn_args* p) { return cut_of(p, parts_of(p, p->dk, p->dv)); }
Cut backward_cut(const hum_decay_attn_args* p) { return cut_of(p, 2 * parts_of(p, p->dv, p->dk) + parts_of(p, p->dk, p->dv)); }

int launched(const char* fn) {
    const hipError_t st = hipGetLastError();
    return st == hipSuccess ? HUM_OK : derr(HUM_ERR_HIP, fn, hipGetErrorString(st));
}

}  // namespace

extern "C" {

int hum_decay_attn_workspace(const hum_decay_attn_args* p, int32_t backward, uint64_t* bytes) {
    const char* fn = "hum_decay_attn_workspace";
    if (const int rc = check_args(fn, p)) return rc;
    if (!bytes) return derr(HUM_ERR_ARG, fn, "null argument");
    *bytes = backward ? 2 * walk_bytes(p, backward_cut(p)) : walk_bytes(p, forward_cut(p));
    if (backward && p->kv_heads != p->heads)   // the heads' partial gradients of shared keys and values
        *bytes += round16(4ull * p->lanes * p->steps * p->heads * p->dk) + 4ull * p->lanes * p->steps * p->heads * p->dv;
    return HUM_OK;
}

int hum_decay_attn(const hum_decay_attn_args* p, const hum_rows* out, void* workspace, uint64_t workspace_bytes, void* stream) {
    const char* fn = "hum_decay_attn";
    if (const int rc = check_args(fn, p)) return rc;
    if (!out || (p->lanes && p->steps && !out->ptr) || ((uintptr_t)out->ptr) % elem_size(p->type))
        return derr(HUM_ERR_ARG, fn, "out is required, aligned to its elements");
    uint64_t need = 0;
    if (const int rc = hum_decay_attn_workspace(p, 0, &need)) return rc;
    if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16))
        return derr(HUM_ERR_ARG, fn, "the workspace is too small (hum_decay_attn_workspace) or not aligned to 16 bytes");
    if (!p->lanes) return HUM_OK;
    const OnDevice dev(p->device);
    if (!dev.ok) return derr(HUM_ERR_HIP, fn, "hipSetDevice");
    const int size = elem_size(p->type), group = p->heads / p->kv_heads;
    Role r = {};
    r.x = rows_of(p->q, 1, size, p->dk);
    r.y = rows_of(p->k, group, size, p->dk);
    r.z = rows_of(p->v, group, size, p->dv);
    r.out = rows_of(*out, 1, size, p->dv);
    r.dy = p->dk;
    r.dz = p->dv;
    r.s_pair = r.s_in = p->scale;
    r.s_add = 1.f;
    role_state(r, p->state_in, p->state_out, p, true);
    const Cut c = forward_cut(p);
    if (c.segs > 1) {
        run_segments(p, r, (float*)workspace, c, (hipStream_t)stream);
        enter_segments(r, (const float*)workspace, p, c);
    }
    launch_roles(p, &r, 1, c, true, (hipStream_t)stream);
    return launched(fn);
}

int hum_decay_attn_backward(const hum_decay_attn_args* p, const hum_rows* d_out, const float* d_state_out,
                            const hum_rows* dq, const hum_rows* dk, const hum_rows* dv, float* d_state_in, void* workspace,
                            uint64_t workspace_bytes, void* stream) {
    const char* fn = "hum_decay_attn_backward";
    if (const int rc = check_args(fn, p)) return rc;
    const hum_rows none = {};
    const hum_rows& gq = dq ? *dq : none;
    const hum_rows& gk = dk ? *dk : none;
    const hum_rows& gv = dv ? *dv : none;
    const int size = elem_size(p->type), group = p->heads / p->kv_heads;
    if (!d_out || (p->lanes && p->steps && !d_out->ptr) || ((uintptr_t)d_out->ptr) % size)
        return derr(HUM_ERR_ARG, fn, "d_out is required, aligned to its elements");
    if (((uintptr_t)gq.ptr | (uintptr_t)gk.ptr | (uintptr_t)gv.ptr) % size || ((uintptr_t)d_state_out | (uintptr_t)d_state_in) % 4)
        return derr(HUM_ERR_ARG, fn, "gradients must be aligned to their elements");
    uint64_t need = 0;
    if (const int rc = hum_decay_attn_workspace(p, 1, &need)) return rc;
    if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16))
        return derr(HUM_ERR_ARG, fn, "the workspace is too small (hum_decay_attn_workspace) or not aligned to 16 bytes");
    const uint64_t state = 4ull * p->lanes * p->heads * p->dk * p->dv;
    auto meets = [&](const float* a, const float* b) {
        return a && b && (uintptr_t)a < (uintptr_t)b + state && (uintptr_t)b < (uintptr_t)a + state;
    };
    if (meets(d_state_in, d_state_out) || meets(d_state_in, p->state_in))
        return derr(HUM_ERR_ARG, fn, "d_state_in must not overlap state_in or d_state_out");
    if (!p->lanes) return HUM_OK;
    const OnDevice dev(p->device);
    if (!dev.ok) return derr(HUM_ERR_HIP, fn, "hipSetDevice");
    const Rows q = rows_of(p->q, 1, size, p->dk), k = rows_of(p->k, group, size, p->dk);
    const Rows v = rows_of(p->v, group, size, p->dv), g = rows_of(*d_out, 1, size, p->dv);
    hipStream_t s = (hipStream_t)stream;
    const Cut c = backward_cut(p);
    float* const seg_s = (float*)workspace;   // segments' states, their gradients, the shared heads' partial gradients
    float* const seg_r = (float*)((char*)seg_s + walk_bytes(p, c));
    float* const part_k = (float*)((char*)seg_r + walk_bytes(p, c));
    float* const part_v = (float*)((char*)part_k + round16(4ull * p->lanes * p->steps * p->heads * p->dk));
    const hum_rows pk = {part_k, (int64_t)p->steps * p->heads * p->dk, (int64_t)p->heads * p->dk, p->dk};
    const hum_rows pv = {part_v, (int64_t)p->steps * p->heads * p->dv, (int64_t)p->heads * p->dv, p->dv};
    Role r[3];
    int n = 0;
    if (gq.ptr) {
        Role& w = r[n++] = Role{};
        w.x = g; w.y = v; w.z = k;
        w.out = rows_of(gq, 1, size, p->dk);
        w.dy = p->dv; w.dz = p->dk;
        w.s_pair = w.s_in = p->scale;
        w.s_add = 1.f;
        role_state(w, p->state_in, nullptr, p, false);
    }
    if (gk.ptr) {
        Role& w = r[n++] = Role{};
        w.x = v; w.y = g; w.z = q;
        w.out = group > 1 ? rows_of(pk, 1, 4, p->dk) : rows_of(gk, 1, size, p->dk);
        w.out_f32 = group > 1;
        w.dy = p->dv; w.dz = p->dk;
        w.rev = 1;
        w.s_pair = w.s_add = p->scale;
        w.s_in = 1.f;
        role_state(w, d_state_out, nullptr, p, false);
    }
    if (gv.ptr || d_state_in) {
        Role& w = r[n++] = Role{};
        w.x = k; w.y = q; w.z = g;
        w.out = gv.ptr ? (group > 1 ? rows_of(pv, 1, 4, p->dv) : rows_of(gv, 1, size, p->dv)) : Rows{};
        w.out.shared = 1;
        w.out_f32 = group > 1;
        w.dy = p->dk; w.dz = p->dv;
        w.rev = 1;
        w.s_pair = w.s_add = p->scale;
        w.s_in = 1.f;
        role_state(w, d_state_out, d_state_in, p, true);
    }
    if (c.segs > 1) {
        Role w = {};
        if (gq.ptr) {
            w.y = k; w.z = v;
            w.dy = p->dk; w.dz = p->dv;
            w.s_add = 1.f;
            role_state(w, p->state_in, nullptr, p, true);
            run_segments(p, w, seg_s, c, s);
        }
        if (gk.ptr || gv.ptr || d_state_in) {
            w = Role{};
            w.y = q; w.z = g;
            w.dy = p->dk; w.dz = p->dv;
            w.rev = 1;
            w.s_add = p->scale;
            role_state(w, d_state_out, nullptr, p, true);
            run_segments(p, w, seg_r, c, s);
        }
        for (int i = 0; i < n; i++) enter_segments(r[i], r[i].rev ? seg_r : seg_s, p, c);
    }
    launch_roles(p, r, n, c, true, s);
    if (group > 1 && p->steps) {
        const long rows = (long)p->lanes * p->steps;
        struct { const hum_rows* o; const float* part; int d; } sums[2] = {{&gk, part_k, p->dk}, {&gv, part_v, p->dv}};
        for (auto& x : sums) {
            if (!x.o->ptr) continue;
            const Rows o = rows_of(*x.o, 1, size, x.d);
            const long blocks = (rows * p->kv_heads * x.d + 255) / 256;
            const dim3 grid((unsigned)(blocks < (1 << 16) ? blocks : (1 << 16)));
            if (p->type == HUM_F32) hipLaunchKernelGGL(share_kernel<HUM_F32>, grid, dim3(256), 0, s, x.part, o, rows, p->steps, p->kv_heads, group, x.d);
            else if (p->type == HUM_BF16) hipLaunchKernelGGL(share_kernel<HUM_BF16>, grid, dim3(256), 0, s, x.part, o, rows, p->steps, p->kv_heads, group, x.d);
            else hipLaunchKernelGGL(share_kernel<HUM_F16>, grid, dim3(256), 0, s, x.part, o, rows, p->steps, p->kv_heads, group, x.d);
        }
    }
    return launched(fn);
}

}  // extern "C"

namespace {
template <int ST, int LPR>
void launch_step_v(const StepArgs& a, bool vec, dim3 grid, hipStream_t s) {
    if (vec) hipLaunchKernelGGL((step_kernel<ST, LPR, true>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((step_kernel<ST, LPR, false>), grid, dim3(256), 0, s, a);
}
template <int ST>
void launch_step(const StepArgs& a, int lpr, bool vec, dim3 grid, hipStream_t s) {
    switch (lpr) {
        case 1: launch_step_v<ST, 1>(a, vec, grid, s); break;
        case 2: launch_step_v<ST, 2>(a, vec, grid, s); break;
        case 4: launch_step_v<ST, 4>(a, vec, grid, s); break;
        case 8: launch_step_v<ST, 8>(a, vec, grid, s); break;
        case 16: launch_step_v<ST, 16>(a, vec, grid, s); break;
        default: launch_step_v<ST, 32>(a, vec, grid, s); break;
    }
}
}  // namespace

extern "C" int hum_decay_attn_step(const hum_decay_attn_args* p, const uint8_t* active, const hum_rows* out, void* stream) {
    const char* fn = "hum_decay_attn_step";
    if (const int rc = check_args(fn, p)) return rc;
    if (p->steps != 1 || p->lengths) return derr(HUM_ERR_ARG, fn, "steps must be 1 and lengths NULL (active says which lanes step)");
    if (!out || (p->lanes && (!out->ptr || !p->state_out)) || ((uintptr_t)out->ptr) % elem_size(p->type))
        return derr(HUM_ERR_ARG, fn, "out (aligned to its elements) and state_out are required");
    if (!p->lanes) return HUM_OK;
    const OnDevice dev(p->device);
    if (!dev.ok) return derr(HUM_ERR_HIP, fn, "hipSetDevice");
    const int size = elem_size(p->type), group = p->heads / p->kv_heads;
    StepArgs a = {};
    a.q = rows_of(p->q, 1, size, p->dk);
    a.k = rows_of(p->k, group, size, p->dk);
    a.v = rows_of(p->v, group, size, p->dv);
    a.out = rows_of(*out, 1, size, p->dv);
    a.log_decay = p->log_decay;
    a.state_in = p->state_in;
    a.state_out = p->state_out;
    a.reset = p->reset;
    a.reset_lane = p->reset_lane;
    a.active = active;
    a.heads = p->heads;
    a.dk = p->dk;
    a.dv = p->dv;
    a.scale = p->scale;
    const bool vec = p->dk % 4 == 0 && ((uintptr_t)p->state_in | (uintptr_t)p->state_out) % 16 == 0;
    int lpr = 1;
    while (4 * lpr < p->dk) lpr *= 2;
    const int rows = 4 * 4 * (64 / lpr);
    a.blocks = (p->dv + rows - 1) / rows;
    const dim3 grid((unsigned)(p->lanes * p->heads * a.blocks));
    if (p->type == HUM_BF16) launch_step<HUM_BF16>(a, lpr, vec, grid, (hipStream_t)stream);
    else if (p->type == HUM_F16) launch_step<HUM_F16>(a, lpr, vec, grid, (hipStream_t)stream);
    else launch_step<HUM_F32>(a, lpr, vec, grid, (hipStream_t)stream);
    return launched(fn);
}
