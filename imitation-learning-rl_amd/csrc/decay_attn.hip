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
// P = (Y X^T) masked and weighted by D, O^T = Z^T P + S^T X^T, S = lambda^32 S + (w Y)^T Z.  A workgroup owns one (lane,
// head); each of its waves owns 32 of z's channels and keeps its slice of S in registers for the whole walk.  The chunk's
// rows come into registers while the chunk before is worked on, and from there into LDS, where all waves read them; P is
// formed by two or four of the waves and shared through LDS.  The rows of every A operand are taken in the order
//     matrix row m of tile a  <->  index 8 (m >> 2) + 4 a + (m & 3)   (of 32)
// under which the accumulators of a pair of tiles (lane group g holds rows 4 g .. 4 g + 3 of each) are exactly the 8
// consecutive contraction indexes 8 g .. 8 g + 7 that lane group needs as an operand of the next product: S feeds O, and P
// goes to the other waves, without a change of layout.  Contractions over the steps read Y and Z back transposed.
//
// What bounds it (bf16, time-major rows).  Many lanes: HBM.  Forward of 4096 lanes x 32 steps, 4 heads x 64 x 64: 0.80 GB
// in 153 us, 5.3 TB/s where a large copy reaches 5.1; gradient 1.28 GB in 298 to 353 us, by which of several equal sets of
// tensors it works on.  Few lanes: the latency of a chunk (LDS
// round trips and dependent matrix instructions), 2 to 4 us of it, since a walk is serial: so walks are cut into segments
// (cut_of), whose states cost traffic of their own.  Forward of 1 x 8192 steps, 8 heads x 128 x 128: segments' states 19,
// scan 13, outputs 30 us.
//
// Rounding.  Every element type goes through the bf16 matrix cores: bf16 inputs as they are, float16 as two bf16 parts and
// float32 as three, exactly but for 2^-27; products of parts are exact in the float32 accumulators.  Computed operands are
// split likewise: P and the state read by O into two parts (2^-18 of the value, under the output's own 2^-9 or 2^-12; three
// for float32), the weighted Z that enters the state into three (2^-27, below float32's 2^-24: the state is held in 32
// bits).  An output is rounded once.  These bounds hold from about 2^-109 on: the matrix cores take parts below 2^-126 as
// zeros (float32 operands of 1e-36 are good to 1e-4), and a float32 from 2^128 - 2^119 on has an infinite first part and
// counts as infinite.
//
// Non-finite values.  A row of Z multiplies zeros of P for the steps that must not see it (earlier steps, other
// episodes, those past which lambda^d is 0), and 0 x inf is NaN: such values of z enter the products as zeros and make NaN of
// the channels of exactly the steps that see them, so an episode that diverged leaves the next one, its own earlier steps
// and what a head without memory does later untouched.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <cstdio>
#include <type_traits>

#include "../../include/humanoid_env.h"
#include "overlap.h"

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
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

struct Rows {               // [lane, step, head, channel] with unit channel stride
    void* p;
    long lane, step, head;  // strides in elements
    int shared;             // heads that read one of its heads
    int near;               // steps lie less than 2^25 bytes apart
    int vec;                // and do not overlap, and rows are of 16-byte units, aligned
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
};

struct WalkArgs {
    Role r[3];
    int nroles;
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

__device__ __forceinline__ f32x8 pair(f32x4 a, f32x4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }
// a * b with 0 times anything 0, infinities and NaN too: a weight of zero is a mask
extern "C" __device__ float mul0(float a, float b) __asm("llvm.amdgcn.fmul.legacy");

// v as N bf16 parts, each the rounding of what the ones before leave
template <int N>
__device__ __forceinline__ void split(f32x8 v, bf16x8 (&o)[N]) {
#pragma unroll
    for (int i = 0; i < N; i++) {
        o[i] = __builtin_convertvector(v, bf16x8);   // to nearest, ties to even
        if (i + 1 < N) {
            const u32x4 u = __builtin_bit_cast(u32x4, o[i]);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                v[2 * j] -= __builtin_bit_cast(float, u[j] << 16);
                v[2 * j + 1] -= __builtin_bit_cast(float, u[j] & 0xffff0000u);
            }
        }
    }
}
template <int N>
__device__ __forceinline__ void split(f32x4 v, bf16x4 (&o)[N]) {
#pragma unroll
    for (int i = 0; i < N; i++) {
        o[i] = __builtin_convertvector(v, bf16x4);
        if (i + 1 < N) {
            const u32x2 u = __builtin_bit_cast(u32x2, o[i]);
#pragma unroll
            for (int j = 0; j < 2; j++) {
                v[2 * j] -= __builtin_bit_cast(float, u[j] << 16);
                v[2 * j + 1] -= __builtin_bit_cast(float, u[j] & 0xffff0000u);
            }
        }
    }
}
template <int N>
__device__ __forceinline__ f32x8 whole(const bf16x8 (&o)[N]) {
    f32x8 v = {};
#pragma unroll
    for (int i = N - 1; i >= 0; i--) {
        const u32x4 u = __builtin_bit_cast(u32x4, o[i]);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float lo = __builtin_bit_cast(float, u[j] << 16), hi = __builtin_bit_cast(float, u[j] & 0xffff0000u);
            v[2 * j] = i == N - 1 ? lo : v[2 * j] + lo;
            v[2 * j + 1] = i == N - 1 ? hi : v[2 * j + 1] + hi;
        }
    }
    return v;
}
// c += a b over 32 contraction indexes; parts i, j with i + j > 2 stay below 2^-27 of the product
template <int NA, int NB>
__device__ __forceinline__ void mma(f32x4& c, const bf16x8 (&a)[NA], const bf16x8 (&b)[NB]) {
#pragma unroll
    for (int i = 0; i < NA; i++)
#pragma unroll
        for (int j = 0; j < NB; j++)
            if (i + j < 3) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[j], c, 0, 0, 0);
}
// rows s0 .. s0 + 7 of 16 columns, 4 neighbours per quarter of 16 lanes, quarters APART: the transposing LDS load
template <int APART>
__device__ __forceinline__ bf16x8 column(const __bf16* m, int pitch, int s0, int c0, int r) {
    typedef __attribute__((address_space(3))) bf16x4 L4;
    const __bf16* p = m + (s0 + (r >> 2)) * pitch + c0 + APART * (r & 3);
    const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((L4*)p);
    const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((L4*)(p + 4 * pitch));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// ---- the element types.  Every one goes through the bf16 matrix cores: a float16 is the sum of two bf16 parts, a float32
// of three, exactly (up to 2^-27), and the product of two such sums takes up to six matrix instructions - 96 cycles where the
// float32 instruction takes 256.  IN: parts of an input, MID: of P and of the state that O reads
template <int ST> struct Num;
template <> struct Num<HUM_BF16> { typedef __bf16 T; static constexpr int IN = 1, MID = 2, SIZE = 2; };
template <> struct Num<HUM_F16> { typedef _Float16 T; static constexpr int IN = 2, MID = 2, SIZE = 2; };
template <> struct Num<HUM_F32> { typedef float T; static constexpr int IN = 3, MID = 3, SIZE = 4; };

// How a walk's rows are accessed.  BUFFER: rows of whole aligned units of 16 bytes, through buffers.  WIDE: 16 bytes at any
// alignment.  ANY: the same with 64-bit addresses and a branch for heads of fewer channels than 16 bytes hold; also steps
// 2^25 bytes apart and more, or backwards in memory.  Gradient of 4096 x 32 steps, 4 heads, bf16: 64 channels in BUFFER
// 300 us, 63 in WIDE 439 (60: 380; the first version, element by element, 916 and 900); WIDE saves 3 % against ANY
enum Mode { BUFFER, WIDE, ANY };

// 16 loaded bytes into the planes of an LDS tile
template <int ST>
__device__ __forceinline__ void put(__bf16* m, int plane, u32x4 raw) {
    if constexpr (ST == HUM_BF16) {
        *(u32x4*)m = raw;
    } else if constexpr (ST == HUM_F16) {
        bf16x8 o[2];
        split<2>(__builtin_convertvector(__builtin_bit_cast(f16x8, raw), f32x8), o);
        *(bf16x8*)m = o[0];
        *(bf16x8*)(m + plane) = o[1];
    } else {
        bf16x4 o[3];
        split<3>(__builtin_bit_cast(f32x4, raw), o);
#pragma unroll
        for (int i = 0; i < 3; i++) *(bf16x4*)(m + i * plane) = o[i];
    }
}
// not 0 where one of 8 values (the first of their parts) is not finite: its exponent is all ones
__device__ __forceinline__ unsigned odd_bits(bf16x8 v) {
    const u32x4 u = __builtin_bit_cast(u32x4, v);
    unsigned bad = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) bad |= (u[i] & 0x7f807f80u) + 0x00800080u;
    return bad & 0x80008000u;
}
// 8 channels of a row, rounded once; bytes `second` on are the upper half of a float32 row's
template <int ST>
__device__ __forceinline__ void store(Buf b, int at, int second, f32x8 v) {
    if constexpr (ST == HUM_F32) {
        buf_store4(b, at, __builtin_shufflevector(v, v, 0, 1, 2, 3));
        buf_store4(b, second, __builtin_shufflevector(v, v, 4, 5, 6, 7));
    } else if constexpr (ST == HUM_F16) {
        buf_store(b, at, __builtin_bit_cast(u32x4, __builtin_convertvector(v, f16x8)));
    } else {
        buf_store(b, at, __builtin_bit_cast(u32x4, __builtin_convertvector(v, bf16x8)));
    }
}

template <int ST>
__device__ __forceinline__ void store(Buf b, int at, int, f32x4 v) {
    if constexpr (ST == HUM_F32) {
        buf_store4(b, at, v);
    } else {
        typedef typename Num<ST>::T E4 __attribute__((ext_vector_type(4)));
        __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, __builtin_convertvector(v, E4)), b, at, 0, 0);
    }
}

// ---- accesses at element alignment (64-bit addresses; the hardware takes 16 bytes at any of them).  A row's last piece must
// not pass the row's end, so it is loaded from an earlier place, where it ends with the row, and shifted down
#define GLOBAL __attribute__((address_space(1)))
typedef unsigned int any4 __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned int any2 __attribute__((ext_vector_type(2), aligned(2)));
typedef unsigned int any1 __attribute__((aligned(2)));
template <typename E> struct Any {
    static constexpr int UNIT = 16 / sizeof(E);
    typedef E V __attribute__((ext_vector_type(UNIT)));
    typedef GLOBAL E* P;
    // UNIT elements of a row of d, from element c on (c may be behind the end): where to load them, and what is loaded
    static __device__ __forceinline__ int place(int c, int d) { return d < UNIT || c < d - UNIT ? c : d - UNIT; }
    static __device__ __forceinline__ u32x4 load(const E* row, int c, int d) {
        const P p = (P)row;
        if (d >= UNIT) return *(GLOBAL any4*)(p + place(c, d));
        V x = {};
#pragma unroll
        for (int j = 0; j < UNIT; j++) x[j] = c + j < d ? p[c + j] : (E)0;   // (a head of few channels)
        return __builtin_bit_cast(u32x4, x);
    }
    // the loaded piece's elements from c - place(c, d) on, zeros behind the row's end
    static __device__ __forceinline__ u32x4 align(u32x4 v, int by) {
        if constexpr (sizeof(E) == 2) {
            const int half = 16 * (by & 1);
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = __builtin_amdgcn_alignbit(i < 3 ? v[i + 1] : 0u, v[i], half);
        }
        const int words = by * (int)sizeof(E) / 4;
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = words & 1 ? (i < 3 ? v[i + 1] : 0u) : v[i];
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = words & 2 ? (i < 2 ? v[i + 2] : 0u) : v[i];
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = words & ~3 ? 0u : v[i];
        return v;
    }
    // the first n (of UNIT, or more for all)
    static __device__ __forceinline__ void store(E* to, int n, u32x4 v) {
        const P p = (P)to;
        if (n >= UNIT) {
            *(GLOBAL any4*)p = v;
            return;
        }
        constexpr int H = UNIT / 2, Q = UNIT / 4;   // elements of 8 bytes, of 4
        if (n & H) *(GLOBAL any2*)p = u32x2{v[0], v[1]};
        const unsigned w0 = n & H ? v[2] : v[0], w1 = n & H ? v[3] : v[1];
        if (n & Q) *(GLOBAL any1*)(p + (n & H)) = w0;
        if constexpr (sizeof(E) == 2) {
            const unsigned short e = (unsigned short)(n & Q ? w1 : w0);
            if (n & 1) p[n & (H + Q)] = __builtin_bit_cast(E, e);
        }
    }
};
template <int ST>
__device__ __forceinline__ void store_some(void* p, long at, int n, f32x4 v) {   // n of 4
    typedef typename Num<ST>::T E;
    E* e = (E*)p + at;
    if constexpr (ST == HUM_F32) {
        Any<E>::store(e, n, __builtin_bit_cast(u32x4, v));
    } else {
        typedef E E4 __attribute__((ext_vector_type(4)));
        const u32x2 u = __builtin_bit_cast(u32x2, __builtin_convertvector(v, E4));
        Any<E>::store(e, n < 4 ? n : 4, u32x4{u[0], u[1], 0, 0});
    }
}
template <int ST>
__device__ __forceinline__ void store_some(void* p, long at, int n, f32x8 v) {   // n of 8 channels, rounded once
    typedef typename Num<ST>::T E;
    E* e = (E*)p + at;
    if constexpr (ST == HUM_F32) {
        Any<E>::store(e, n, __builtin_bit_cast(u32x4, __builtin_shufflevector(v, v, 0, 1, 2, 3)));
        if (n > 4) Any<E>::store(e + 4, n - 4, __builtin_bit_cast(u32x4, __builtin_shufflevector(v, v, 4, 5, 6, 7)));
    } else {
        typedef E E8 __attribute__((ext_vector_type(8)));
        Any<E>::store(e, n, __builtin_bit_cast(u32x4, __builtin_convertvector(v, E8)));
    }
}

// what the workgroup's waves wrote to LDS before it, all of them read behind it (loads in flight stay in flight)
template <int WAVES>
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    if constexpr (WAVES > 1) __builtin_amdgcn_s_barrier();
    else __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
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

// waves per SIMD that the registers are limited for (the state takes 16 K of them): the most that fit without scratch memory,
// a few bytes of which cost more than a wave gives (4096 x 32 steps, 4 heads x 64 x 64, bf16: 156 us and gradient 300 with
// three waves, 175 and 379 with two, 228 and 509 with four and their scratch)
constexpr int walk_waves(int st, int k, int w, Mode mode) {   // (a single wave has all of a chunk's rows in flight)
    const bool alone = k > 1 && w == 1;
    if (mode != BUFFER) return st == HUM_BF16 ? (k > 1 ? 2 : 3) : k > 2 ? 1 : 2;
    return st == HUM_BF16 ? (k > 2 && alone ? 1 : k > 2 || alone ? 2 : 3) : st == HUM_F16 ? (k > 2 && alone ? 1 : 2) : k > 2 || alone ? 1 : 2;
}

// One workgroup per HEADS neighbouring heads of a lane, role and segment; W waves per head, each with 32 of z's channels and
// its slice of the state.  A head's waves share the chunk's x and y rows (K operands of 32 channels) and P; the heads of a
// workgroup only share the loading, so that a load meets long pieces of few rows (with one head, 4096 lanes' time-major
// steps lie 2 MB apart and each load meets 8 pages for 1 KB: forward 168 us, 156 us with the heads together).  OUTS: rows
// come out (else the states of the segments are wanted only).
template <int ST, int K, int W, int J, int HEADS, Mode MODE, bool OUTS>
__global__ void __launch_bounds__(64 * W * HEADS, walk_waves(ST, K, W, MODE)) walk_kernel(WalkArgs a) {
    constexpr int IN = Num<ST>::IN, MID = Num<ST>::MID, SIZE = Num<ST>::SIZE, UNIT = 16 / SIZE;
    constexpr int D = 32 * K;                  // channels of x and y rounded up
    constexpr int PITCH = D + 8;               // of x and y in LDS: 16-byte reads of 16 rows meet no bank twice
    constexpr int Z = 16 * J;                  // channels of z of a wave
    constexpr int PLANE = CH * PITCH, ZPLANE = CH * Z;
    constexpr int T = 64 * W * HEADS, B = W * HEADS;   // threads, waves
    __shared__ __attribute__((aligned(16))) __bf16 tx[HEADS][OUTS ? IN * PLANE : 8], ty[HEADS][IN * PLANE], tz[HEADS][W][IN * ZPLANE];
    __shared__ __attribute__((aligned(16))) bf16x8 tp[HEADS][OUTS ? 2 : 1][MID][64];
    // lambda^d times the scale's part for d = -31 .. 32 steps, zeros for d < 0: between two steps of a chunk, and from a
    // step to the chunk's end
    __shared__ float pows_pair[HEADS][2 * CH], pows_add[HEADS][2 * CH];
    __shared__ unsigned odds[HEADS][W][Z];

    const int tid = threadIdx.x, l = tid & 63, g = l >> 4, r = l & 15;
    const int sub = HEADS > 1 ? __builtin_amdgcn_readfirstlane(tid / (64 * W)) : 0;   // the wave's head of the workgroup's
    const int wave = __builtin_amdgcn_readfirstlane(tid / 64 % W);                     // and its channels of z
    __bf16 *const lx = tx[sub], *const ly = ty[sub], *const lz = tz[sub][wave];
    bf16x8(*const lp)[MID][64] = tp[sub];
    float *const pow_pair = pows_pair[sub], *const pow_add = pows_add[sub];
    unsigned* const lodd = odds[sub][wave];
    // the roles of one segment read the same rows, and NEAR segments in a row are neighbours in memory (the heads of a lane,
    // lanes of a time-major step): they go to one XCD, one after the other.  Gradient of 4096 lanes x 32 steps, bf16,
    // 3 heads x 64 x 64: 212 us, 231 with NEAR = 1, 211 with 32 (which leaves XCDs idle at few lanes); 4 heads, which share a
    // workgroup, 300 with any
    const int block = blockIdx.x, ri = block / XCDS % a.nroles, turn = block / (XCDS * a.nroles);
    const int item = (turn / NEAR * XCDS + block % XCDS) * NEAR + turn % NEAR;
    if (item >= a.lanes * a.heads / HEADS * a.segs) return;
    const int group = item / a.segs, seg = item - group * a.segs;
    const Role& R = a.r[ri];
    const int dz0 = Z * wave;
    const int b = group * HEADS / a.heads, h0 = group * HEADS - b * a.heads, h = h0 + sub, unit = b * a.heads + h;
    const int steps = a.steps;
    int len = steps;
    if (a.lengths) {
        len = __builtin_amdgcn_readfirstlane(a.lengths[b]);
        len = len < 0 ? 0 : len > steps ? steps : len;
    }
    const int rev = R.rev, dy = R.dy, dz = R.dz;
    const float lg = a.log_decay[h] * 1.44269504088896340736f;
    auto power = [&](int n) { return n == 0 ? 1.f : __builtin_amdgcn_exp2f(lg * (float)n); };
    if (wave == 0) {
        pow_pair[l] = l < CH - 1 ? 0.f : R.s_pair * power(l - (CH - 1));
        pow_add[l] = l < CH - 1 ? 0.f : R.s_add * power(l - (CH - 1));
    }
    // a step is seen for `reach` steps, itself among them; then its weight lambda^d is 0 in float32 (33: as far as a chunk and
    // the state behind it ask).  A weight of 0 is a mask, also for what is not finite: see `leaving`.  fades: of any head of
    // the workgroup's, since barriers hang on it
    const int reach = __popcll(__ballot(l <= CH && power(l) != 0.f));
    bool fades = HEADS == 1 && reach <= CH;
    if constexpr (HEADS > 1)
        for (int i = 0; i < HEADS; i++) fades |= __builtin_amdgcn_exp2f(a.log_decay[h0 + i] * 1.44269504088896340736f * (float)CH) == 0.f;
    const int seg0 = seg * a.seg_steps, seg1 = seg + 1 < a.segs ? seg0 + a.seg_steps : steps;
    const int end = len < seg1 ? len : seg1;
    auto row_of = [&](int tile) { return 8 * (r >> 2) + 4 * tile + (r & 3); };
    auto time = [&](int n) { return rev ? len - 1 - n : n; };   // of walk step n
    auto head_of = [&](const Rows& m, int head) { return (long)b * m.lane + (long)(head / m.shared) * m.head; };

    // ---- rows of a chunk: x and y by all waves, z by each wave its channels, in units of 16 bytes along a row: unit u of
    // thread t is unit t % PER of row u T / PER + t / PER.  BUFFER: a chunk of L steps is a buffer from its earliest time to its
    // last row's end, so the steps behind L lie outside (walking backwards: before it, at negative offsets, which are
    // large ones); `at` is the address of the walk's next chunk's first row
    struct View {
        const char* at;
        long hop;       // to the next chunk
        int step, row;  // bytes from walk step to walk step forwards in time, bytes of a row
        int off;        // the thread's byte offset
    };
    const int dir = rev ? -1 : 1;
    auto view = [&](const Rows& m, int size, int d, int row, int head, int channel) {   // head: of the workgroup's
        auto place = [&](int i) { return HEADS > 1 ? ((h0 + i) / m.shared - h0 / m.shared) * (int)m.head * size : 0; };
        View v;
        v.step = (int)m.step * size;
        v.at = (const char*)m.p + (head_of(m, h0) + (long)time(seg0) * m.step) * size;
        v.hop = (long)dir * CH * v.step;
        v.row = place(HEADS - 1) + d * size;
        v.off = channel < d && row < CH ? dir * row * v.step + place(head) + channel * size : OUTSIDE;   // (8 waves load 64 rows)
        return v;
    };
    auto chunk = [&](const View& v, int L) { return buffer(rev ? v.at - (long)(L - 1) * v.step : v.at, (L - 1) * v.step + v.row); };
    constexpr int PER = D / UNIT, PERZ = Z * W / UNIT;               // units of a head's row of x and y, of z
    constexpr int ROWS = T / (HEADS * PER), ROWSZ = T / (HEADS * PERZ);   // rows of a load
    constexpr int N = ROWS < CH ? CH / ROWS : 1, NZ = CH / ROWSZ;         // loads of a thread
    const int in_row = tid % (HEADS * PER), in_rowz = tid % (HEADS * PERZ), row = tid / (HEADS * PER), rowz = tid / (HEADS * PERZ);
    View vx = {}, vy = {}, vz = {}, vo = {};
    const int out_size = R.out_f32 ? 4 : SIZE;
    const unsigned char* marks = a.reset ? a.reset + (long)b * a.reset_lane : nullptr;
    const char* at_mark = nullptr;
    const int mark_step = (int)a.reset_step, mark_off = (rev ? 1 - l : l) * mark_step;
    if constexpr (MODE == BUFFER) {
        vy = view(R.y, SIZE, dy, row, in_row / PER, in_row % PER * UNIT);
        vz = view(R.z, SIZE, dz, rowz, in_rowz / PERZ, in_rowz % PERZ * UNIT);
        if constexpr (OUTS) {
            vx = view(R.x, SIZE, dy, row, in_row / PER, in_row % PER * UNIT);
            vo = view(R.out, out_size, dz, r, sub, dz0 + 4 * J * g);
        }
        at_mark = marks ? (const char*)marks + (long)time(seg0) * a.reset_step : nullptr;
    }
    u32x4 rx[OUTS ? N : 1], ry[N], rz[NZ];
    int mark = 0;
    auto fetch = [&](const Rows& m, View& v, int rows, int row, int channel, int d, int n0, int L, auto& raw) {   // (HEADS 1 if not BUFFER)
        constexpr int M = sizeof(raw) / 16;
        if constexpr (MODE == BUFFER) {
            const Buf bm = chunk(v, L);
            const int base = rev ? (L - 1) * v.step : 0;
#pragma unroll
            for (int u = 0; u < M; u++) raw[u] = buf_load(bm, v.off + (base + dir * u * rows * v.step));
            v.at += v.hop;
        } else {
            // (a row behind the chunk's last step loads the last one's: it is made zeros)
            typedef typename Num<ST>::T E;
            const GLOBAL char* base = (const GLOBAL char*)m.p + (head_of(m, h) + (long)time(n0 + (rev ? L - 1 : 0)) * m.step) * SIZE;
#pragma unroll
            for (int u = 0; u < M; u++) {
                const int n = u * rows + row, k = n < L ? n : L - 1, t = rev ? L - 1 - k : k;
                if constexpr (MODE == WIDE) raw[u] = *(const GLOBAL any4*)(base + (unsigned)(t * (int)m.step + Any<E>::place(channel, d)) * SIZE);
                else raw[u] = Any<E>::load((const E*)(const char*)base + t * m.step, channel, d);
            }
        }
    };
    auto load_rows = [&](int n0) {
        const int L = end - n0 < CH ? end - n0 : CH;
        if constexpr (OUTS) fetch(R.x, vx, ROWS, row, in_row * UNIT, dy, n0, L, rx);
        fetch(R.y, vy, ROWS, row, in_row * UNIT, dy, n0, L, ry);
        fetch(R.z, vz, ROWSZ, rowz, in_rowz * UNIT, dz, n0, L, rz);
        // lane j has the mark that separates the chunk's walk steps j - 1 and j (0: from the entering state, L: from the
        // leaving one).  An episode's first step is cut off from what time puts before it, so the backward walk has it one
        // later.
        if constexpr (MODE == BUFFER) {
            const Buf bm = buffer(rev ? at_mark - (long)(L - 1) * mark_step : at_mark, marks ? (L - 1) * mark_step + 1 : 0);
            mark = __builtin_amdgcn_raw_buffer_load_b8(bm, mark_off + (rev ? (L - 1) * mark_step : 0), 0, 0);
            at_mark += (long)dir * CH * mark_step;
        } else if (marks) {
            const int n = l - rev;   // (lanes outside the chunk's steps are not asked)
            mark = marks[(long)time(n0 + (n < 0 ? 0 : n < L ? n : L - 1)) * a.reset_step];
        }
    };
    auto lay = [&](__bf16* m, int pitch, int plane, int rows, int row, int channel, int d, int L, int at, const auto& raw) {
        constexpr int M = sizeof(raw) / 16;
        typedef Any<typename Num<ST>::T> A;
#pragma unroll
        for (int u = 0; u < M; u++)
            if (u * rows + row < CH) {
                u32x4 v = raw[u];
                if constexpr (MODE != BUFFER) {
                    v = A::align(v, channel - A::place(channel, d));
                    v = u * rows + row < L ? v : u32x4{0, 0, 0, 0};
                }
                put<ST>(m + (u * rows + row) * pitch + at, plane, v);
            }
    };
    if (seg0 < end) load_rows(seg0);

    // ---- the entering state: tile (i, j) holds y channels 32 (i / 2) + 8 g + 4 (i & 1) + 0..3 of z channel zc(j)
    f32x4 S[2 * K][J];
    auto zc = [&](int j) { return dz0 + 4 * J * (r >> 2) + 4 * j + (r & 3); };
    // rows of unit stride are read 16 bytes at a time: along y directly, along z by one row a quad lane and a transpose
    const bool along_y = R.sy == 1;
    const int quad = along_y ? 0 : r & 3, s_y = along_y ? 1 : dz, s_z = along_y ? dy : 1;
    auto state_at = [&](int i, int j) {   // byte offset of a tile's 16 bytes
        const int y = 32 * (i >> 1) + 8 * g + 4 * (i & 1) + quad, z = zc(j) - quad;
        return 4 * (__mul24(z, s_z) + __mul24(y, s_y)) | beyond(y, dy) | beyond(z, dz);
    };
    const int s_d = along_y ? dy : dz;
    auto state_piece = [&](int i, int j, int& c, bool& in) {   // the element of the row of unit stride it begins at, and which row
        const int y = 32 * (i >> 1) + 8 * g + 4 * (i & 1) + quad, z = zc(j) - quad;
        const int row = along_y ? z : y, rows = along_y ? dz : dy;
        c = along_y ? y : z;
        in = row < rows;
        return (in ? row : rows - 1) * s_d;
    };
    auto turn_state = [&] {
        if (!along_y)
#pragma unroll
            for (int j = 0; j < J; j++)
#pragma unroll
                for (int i = 0; i < 2 * K; i++) S[i][j] = quad_transpose(S[i][j]);
    };
    {
        const float* s = R.state_in ? R.state_in + (long)unit * R.in_unit + (long)seg * R.in_seg : nullptr;
        if constexpr (MODE == BUFFER) {
            const Buf bs = buffer(s, 4 * dy * dz);
#pragma unroll
            for (int j = 0; j < J; j++)
#pragma unroll
                for (int i = 0; i < 2 * K; i++) S[i][j] = buf_load4(bs, state_at(i, j));
            turn_state();
        } else {
            typedef Any<float> A;
#pragma unroll
            for (int j = 0; j < J; j++)
#pragma unroll
                for (int i = 0; i < 2 * K; i++) {
                    int c;
                    bool in;
                    const int at = state_piece(i, j, c, in);
                    S[i][j] = s ? __builtin_bit_cast(f32x4, A::load(s + at, c, s_d)) : f32x4{0.f, 0.f, 0.f, 0.f};
                }
#pragma unroll
            for (int j = 0; j < J; j++)
#pragma unroll
                for (int i = 0; i < 2 * K; i++) {
                    int c;
                    bool in;
                    state_piece(i, j, c, in);
                    const u32x4 v = A::align(__builtin_bit_cast(u32x4, S[i][j]), c - A::place(c, s_d));
                    S[i][j] = in ? __builtin_bit_cast(f32x4, v) : f32x4{0.f, 0.f, 0.f, 0.f};
                }
            turn_state();
        }
    }
    float w_in[2];
#pragma unroll
    for (int c = 0; c < 2; c++) w_in[c] = R.s_in * power(16 * c + r + 1 - rev);
    float passed = 1.f;   // what is left of the entering state
    // everything loaded so far (vmcnt 0): else each use of the state in the loop would wait for the next chunk's rows too,
    // which the compiler cannot tell from the state's own loads
    __builtin_amdgcn_s_waitcnt(0x0f70);

    for (int n0 = seg0; n0 < end; n0 += CH) {
        const int L = end - n0 < CH ? end - n0 : CH;
        const bool more = n0 + CH < end;
        // a mark behind the chunk's last step (lane L's, walking backwards) is this chunk's as well as the next one's first
        const unsigned long long cut = __ballot(mark != 0) & ((2ull << (L - 1 + rev)) - 1) & ~(unsigned long long)rev;
        // the last cut at or before step n of the chunk: step n sees the steps from there on, and what entered the chunk only
        // if there is none
        auto cuts_to = [&](int n) { return cut & ((2ull << n) - 1); };
        auto last_cut = [&](unsigned long long m) { return m ? 63 - __builtin_clzll(m) : 0; };
        const int kept = last_cut(cut), faded = L + rev - reach;
        const int leaving = kept > faded ? kept : faded;   // what leaves the chunk is of the steps from here on

        lds_barrier<B>();   // the chunk before has been read
        if constexpr (OUTS) lay(tx[in_row / PER], PITCH, PLANE, ROWS, row, in_row * UNIT, dy, L, in_row % PER * UNIT, rx);
        lay(ty[in_row / PER], PITCH, PLANE, ROWS, row, in_row * UNIT, dy, L, in_row % PER * UNIT, ry);
        // (each wave's channels of z have a tile of their own)
        lay(tz[in_rowz / PERZ][in_rowz % PERZ * UNIT / Z], Z, ZPLANE, ROWSZ, rowz, in_rowz * UNIT, dz, L, in_rowz * UNIT % Z, rz);
        lds_barrier<B>();
        if (more) load_rows(n0 + CH);   // the chunk is in LDS: the registers take the next one's rows
        auto read = [&](const __bf16* m, int row, int k, bf16x8 (&o)[IN]) {
#pragma unroll
            for (int i = 0; i < IN; i++) o[i] = *(const bf16x8*)(m + i * PLANE + row * PITCH + 32 * k + 8 * g);
        };

        // ---- P^T: rows s (step row_of(t)), columns t (walk step 16 c + r).  Tile (t, c) is formed by wave 2 c + t for all
        // where slices are thin and there are as many, else both of a column by wave c (or the only one)
        if constexpr (OUTS) {
            constexpr bool QUARTERS = J == 1 && W >= 4;
            constexpr int NT = QUARTERS ? 1 : 2;
#pragma unroll
            for (int c = 0; c < 2; c++) {
                if (W > 1 && (QUARTERS ? wave >> 1 : wave) != c) continue;
                const int t0 = QUARTERS ? wave & 1 : 0;
                f32x4 p[NT];
#pragma unroll
                for (int t = 0; t < NT; t++) p[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < K; k++) {
                    bf16x8 x[IN], y[IN];
                    read(lx, 16 * c + r, k, x);
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        read(ly, row_of(t0 + t), k, y);
                        mma(p[t], y, x);
                    }
                }
                float w[4 * NT];
#pragma unroll
                for (int j = 0; j < 4 * NT; j++) w[j] = pow_pair[CH - 1 + 16 * c + r - 8 * g - 4 * t0 - j];
                if (cut) {
                    const int seen = last_cut(cuts_to(16 * c + r)) - 8 * g - 4 * t0;
#pragma unroll
                    for (int j = 0; j < 4 * NT; j++) w[j] = j >= seen ? w[j] : 0.f;
                }
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int j = 0; j < 4; j++) p[t][j] = mul0(p[t][j], w[4 * t + j]);
                if constexpr (QUARTERS) {
                    bf16x4 parts[MID];
                    split(p[0], parts);
#pragma unroll
                    for (int u = 0; u < MID; u++) ((bf16x4*)&lp[c][u][l])[t0] = parts[u];
                } else {
                    bf16x8 parts[MID];
                    split(pair(p[0], p[1]), parts);
#pragma unroll
                    for (int u = 0; u < MID; u++) lp[c][u][l] = parts[u];
                }
            }
            lds_barrier<B>();
        }
        if (kept > 0 || fades) {   // z's weights will be zeros for these steps, which a y row that is not finite would not heed
            for (int e = tid % (64 * W); e < leaving * IN * (D / 8); e += 64 * W) {
                const int row = e / (IN * (D / 8)), at = e % (IN * (D / 8));
                *(u32x4*)(ly + at / (D / 8) * PLANE + row * PITCH + at % (D / 8) * 8) = u32x4{0, 0, 0, 0};
            }
            lds_barrier<B>();
        }

        __builtin_amdgcn_sched_barrier(0);   // (what the scheduler would move across costs more registers than there are)
        if (dz0 < dz) {   // a wave behind z's channels only helps to load
            bf16x8 T[J][IN];   // Z^T
#pragma unroll
            for (int j = 0; j < J; j++)
#pragma unroll
                for (int i = 0; i < IN; i++) T[j][i] = column<4 * J>(lz + i * ZPLANE, Z, 8 * g, 4 * j, r);
            // z values that are not finite: zeros to the products, and NaN to what sees them.  The steps at which a channel
            // has some go to odd[channel]
            unsigned odd[J] = {};
            const bool slow = __any((odd_bits(T[0][0]) | odd_bits(T[J - 1][0])) != 0);
            if (slow) {
#pragma unroll
                for (int j = 0; j < J; j++) {
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const bool is = (__builtin_bit_cast(unsigned short, (__bf16)T[j][0][e]) & 0x7f80) == 0x7f80;
                        odd[j] |= is ? 1u << (8 * g + e) : 0u;
#pragma unroll
                        for (int i = 0; i < IN; i++) T[j][i][e] = is ? (__bf16)0.f : T[j][i][e];
                    }
                    odd[j] |= __shfl_xor(odd[j], 16);
                    odd[j] |= __shfl_xor(odd[j], 32);
                    if (g == 0) lodd[4 * J * (r >> 2) + 4 * j + (r & 3)] = odd[j];
                }
                lds_barrier<1>();
            }
            // O^T: rows z channels, columns t
            if constexpr (OUTS) {
                f32x4 o[2][J];
#pragma unroll
                for (int c = 0; c < 2; c++)
#pragma unroll
                    for (int j = 0; j < J; j++) o[c][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < K; k++) {
                    bf16x8 x[2][IN];
                    read(lx, r, k, x[0]);
                    read(lx, 16 + r, k, x[1]);
#pragma unroll
                    for (int j = 0; j < J; j++) {
                        bf16x8 sp[MID];
                        split(pair(S[2 * k][j], S[2 * k + 1][j]), sp);
#pragma unroll
                        for (int c = 0; c < 2; c++) mma(o[c][j], sp, x[c]);
                    }
                }
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    const int n = 16 * c + r, d = dz0 + 4 * J * g;
                    float wi = w_in[c];
                    if (cut) wi = cuts_to(n) ? 0.f : wi;
                    bf16x8 P[MID];
#pragma unroll
                    for (int u = 0; u < MID; u++) P[u] = lp[c][u][l];
#pragma unroll
                    for (int j = 0; j < J; j++) {
#pragma unroll
                        for (int q = 0; q < 4; q++) o[c][j][q] = mul0(o[c][j][q], wi);
                        mma(o[c][j], T[j], P);
                    }
                    if (slow) {
                        const int from = last_cut(cuts_to(n)), near = n + 1 - reach;
                        const unsigned sees = ((2u << n) - 1) & ~((1u << (from > near ? from : near)) - 1);
#pragma unroll
                        for (int j = 0; j < J; j++)
#pragma unroll
                            for (int q = 0; q < 4; q++)
                                if (lodd[4 * J * g + 4 * j + q] & sees) o[c][j][q] = __builtin_nanf("");
                    }
                    auto joined = [&] {
                        if constexpr (J == 1) return o[c][0];
                        else return pair(o[c][0], o[c][1]);
                    };
                    const auto v = joined();
                    if constexpr (MODE == BUFFER) {
                        const Buf bo = buffer(R.out.p ? (rev ? vo.at - (long)(L - 1) * vo.step : vo.at) : nullptr, (L - 1) * vo.step + vo.row);
                        int at = vo.off + ((rev ? (L - 1) * vo.step : 0) + dir * 16 * c * vo.step);
                        const int second = (at + 16) | beyond(d + 4, dz);
                        if (ST == HUM_F32 || R.out_f32) store<HUM_F32>(bo, at, second, v);
                        else store<ST>(bo, at, second, v);
                    } else if (R.out.p && n < L && d < dz) {
                        const long at = head_of(R.out, h) + (long)time(n0 + n) * R.out.step + d;
                        if (R.out_f32) store_some<HUM_F32>(R.out.p, at, dz - d, v);
                        else store_some<ST>(R.out.p, at, dz - d, v);
                    }
                }
            }
            // the state behind the chunk (rows behind the chunk's last step are zeros)
            __builtin_amdgcn_sched_barrier(0);
            if (more || R.state_out) {
                const float through = cut ? 0.f : power(L);
                passed *= through;
#pragma unroll
                for (int i = 0; i < 2 * K; i++)
#pragma unroll
                    for (int j = 0; j < J; j++)
#pragma unroll
                        for (int q = 0; q < 4; q++) S[i][j][q] = mul0(S[i][j][q], through);
                float w[8];
#pragma unroll
                for (int j = 0; j < 8; j++) w[j] = pow_add[CH - 1 + L - 1 + rev - 8 * g - j];
                if (cut)
#pragma unroll
                    for (int j = 0; j < 8; j++) w[j] = 8 * g + j >= leaving ? w[j] : 0.f;
                bf16x8 zp[J][3];
#pragma unroll
                for (int j = 0; j < J; j++) {
                    f32x8 v = whole(T[j]);
#pragma unroll
                    for (int q = 0; q < 8; q++) v[q] = mul0(v[q], w[q]);
                    split(v, zp[j]);
                }
#pragma unroll
                for (int i = 0; i < 2 * K; i++) {
                    bf16x8 y[IN];
#pragma unroll
                    for (int u = 0; u < IN; u++) y[u] = column<8>(ly + u * PLANE, PITCH, 8 * g, 32 * (i >> 1) + 4 * (i & 1), r);
#pragma unroll
                    for (int j = 0; j < J; j++) mma(S[i][j], y, zp[j]);
                }
                if (slow) {
                    const unsigned sees = (unsigned)((1ull << L) - 1) & ~(unsigned)((1ull << leaving) - 1);
#pragma unroll
                    for (int j = 0; j < J; j++)
                        if (odd[j] & sees)
#pragma unroll
                            for (int i = 0; i < 2 * K; i++)
#pragma unroll
                                for (int q = 0; q < 4; q++) S[i][j][q] = __builtin_nanf("");
                }
            }
        }
        if constexpr (MODE == BUFFER && OUTS) vo.at += vo.hop;
    }

    // ---- the steps behind the lane's length
    typedef typename std::conditional<J == 1, f32x4, f32x8>::type Zero;
    if (OUTS && R.out.p && dz0 + 4 * J * g < dz)
        for (int n = (len > seg0 ? len : seg0) + r; n < seg1; n += 16) {
            const int d = dz0 + 4 * J * g;
            const long at = head_of(R.out, h) + (long)n * R.out.step + d;
            if (R.out_f32) store_some<HUM_F32>(R.out.p, at, dz - d, Zero{});
            else store_some<ST>(R.out.p, at, dz - d, Zero{});
        }
    if (R.through && wave == 0 && l == 0) R.through[unit * a.segs + seg] = passed;
    if (R.state_out && (!a.last_only || seg + 1 == a.segs)) {
        float* s = R.state_out + (long)unit * R.out_unit + (long)seg * R.out_seg;
        if constexpr (MODE == BUFFER) {
            const Buf bs = buffer(s, 4 * dy * dz);
            turn_state();
#pragma unroll
            for (int j = 0; j < J; j++)
#pragma unroll
                for (int i = 0; i < 2 * K; i++) buf_store4(bs, state_at(i, j), S[i][j]);
        } else {
            turn_state();
#pragma unroll
            for (int j = 0; j < J; j++)
#pragma unroll
                for (int i = 0; i < 2 * K; i++) {
                    int c;
                    bool in;
                    const int at = state_piece(i, j, c, in);
                    if (in && c < s_d) Any<float>::store(s + at + c, s_d - c, __builtin_bit_cast(u32x4, S[i][j]));
                }
        }
    }
}

// the segments' entering states from what each of them adds: seg[g] <- state before segment g, one thread per element of
// walk blockIdx.y.  A recurrence over the segments that only their loads' latency bounds: AHEAD of them are in flight
// (64 segments of 8 heads x 128 x 128: 13 us, 22 us with 8 in flight of 16 bytes each)
struct ScanArgs {
    struct { const float* in; float* seg; const float* through; } w[2];
    int segs, size;
    long units;
};
__global__ void __launch_bounds__(256) scan_kernel(ScanArgs a) {
    constexpr int AHEAD = 32;
    const long e = (long)blockIdx.x * 256 + threadIdx.x;
    if (e >= a.units * a.size) return;
    const auto& w = a.w[blockIdx.y];
    const int segs = a.segs;
    const long unit = e / a.size, size = a.size;
    float cur = w.in ? w.in[e] : 0.f;
    float* s = w.seg + unit * segs * size + (e - unit * size);
    const float* th = w.through + unit * segs;
    for (int g0 = 0; g0 < segs; g0 += AHEAD) {
        float add[AHEAD], t[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {   // (the last segment's own is not needed)
            const int g = g0 + i < segs ? g0 + i : segs - 1;
            add[i] = s[g * size];
            t[i] = th[g];
        }
#pragma unroll
        for (int i = 0; i < AHEAD; i++)
            if (g0 + i < segs) {
                s[(g0 + i) * size] = cur;
                cur = mul0(cur, t[i]) + add[i];   // behind a cut (t 0) nothing of the old state is left
            }
    }
}

// gradients of keys (blockIdx.y 0) and values (1) that `group` heads share: the sum of the heads' float32 partial results
// part [lanes, steps, heads, d] -> out [lanes, steps, heads / group, d]; one thread per output channel, the heads in order
// (21 lanes x 131 steps, 4 heads to 1: 4 us, a launch's latency)
struct ShareArgs {
    struct { const float* part; Rows out; int d; } x[2];
    long rows;
    int steps, kv, group;
};
template <int ST>
__global__ void __launch_bounds__(256) share_kernel(ShareArgs a) {
    const auto& x = a.x[blockIdx.y];
    const int d = x.d, kv = a.kv, group = a.group;
    if (!x.out.p) return;
    for (long e = (long)blockIdx.x * 256 + threadIdx.x; e < a.rows * kv * d; e += (long)gridDim.x * 256) {
        const long row = e / d, bt = row / kv;   // (lane, step, kv head), (lane, step)
        const int c = (int)(e - row * d), g = (int)(row - bt * kv);
        float s = 0.f;
        for (int i = 0; i < group; i++) s += x.part[((bt * kv + g) * group + i) * d + c];
        const long at = bt / a.steps * x.out.lane + bt % a.steps * x.out.step + (long)g * x.out.head + c;
        ((typename Num<ST>::T*)x.out.p)[at] = (typename Num<ST>::T)s;
    }
}

// ---- single step: S = a S + v k^T, o = scale S q, all in float32 on the vector units - the state is read and written
// once (8 bytes for 4 operations), so HBM bounds it.  LPR lanes of 4 key channels hold one row of S; a wave has
// 64 / LPR rows in one load and U loads in flight, issued before anything that decides whether they are used.  4096 lanes,
// 4 heads x 64 x 64: 0.55 GB in 93 us, 5.8 TB/s; one lane: 10 us, the host's.
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

// A row's last piece of 4 channels is the row's last 4: the lane does what its neighbour does to the channels before its own
// (both store the same) and leaves them out of its sum.  Buffers take 16 bytes at any multiple of 4.  (One lane per row:
// single channels, as there may be fewer than 4.)
template <int ST, int LPR>
__global__ void __launch_bounds__(256) step_kernel(StepArgs a) {
    constexpr int U = 4, ROWS = 64 / LPR;
    const int unit = blockIdx.x / a.blocks, blk = blockIdx.x - unit * a.blocks;
    const int b = unit / a.heads, h = unit - b * a.heads;
    const int wave = threadIdx.x >> 6, l = threadIdx.x & 63;
    const int own = 4 * (l % LPR), c0 = LPR == 1 || own + 4 <= a.dk ? own : a.dk - 4, row0 = (blk * 4 + wave) * U * ROWS + l / LPR;
    const long size = (long)a.dv * a.dk;
    const Buf si = buffer(a.state_in ? a.state_in + unit * size : nullptr, 4 * (int)size), so = buffer(a.state_out + unit * size, 4 * (int)size);
    int at[U];   // byte offsets of a lane's first channel
    f32x4 s[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int row = row0 + u * ROWS;
        at[u] = 4 * (__mul24(row, a.dk) + c0) | beyond(row, a.dv) | beyond(own, a.dk);
        if constexpr (LPR > 1) {
            s[u] = buf_load4(si, at[u]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++)
                s[u][j] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(si, (at[u] + 4 * j) | beyond(j, a.dk), 0, 0));
        }
    }
    const long qo = (long)b * a.q.lane + (long)(h / a.q.shared) * a.q.head, ko = (long)b * a.k.lane + (long)(h / a.k.shared) * a.k.head;
    const long vo = (long)b * a.v.lane + (long)(h / a.v.shared) * a.v.head, oo = (long)b * a.out.lane + (long)h * a.out.head;
    float q[4], k[4], v[U];
#pragma unroll
    for (int j = 0; j < 4; j++) {   // (a channel behind the last reads the last: it is not stored)
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
    const bool forget = fresh || lambda == 0.f;   // (0 times what is not finite)
    const bool keep = !on && a.state_in == a.state_out;   // an idle lane's state in place stays as it is
    float o[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        o[u] = 0.f;
        if (on) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const bool in = LPR > 1 ? c0 + j >= own : j < a.dk;
                s[u][j] = (forget ? 0.f : s[u][j] * lambda) + v[u] * k[j];
                o[u] += in ? s[u][j] * q[j] : 0.f;
            }
            o[u] = row_sum<LPR>(o[u]) * a.scale;
        }
        if (!keep) {
            if constexpr (LPR > 1) {
                buf_store4(so, at[u], s[u]);
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++)
                    __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, (float)s[u][j]), so, (at[u] + 4 * j) | beyond(j, a.dk), 0, 0);
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
    const bool near = r.step >= 0 && r.step < (1l << 25) / size;
    const bool vec = ((uintptr_t)r.ptr | (uintptr_t)(r.lane * size) | (uintptr_t)(r.step * size) | (uintptr_t)(r.head * size)) % 16 == 0 &&
                     d * size % 16 == 0 && r.step >= d && near;
    return Rows{r.ptr, (long)r.lane, (long)r.step, (long)r.head, shared, near, vec};
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

// the memory that arguments stand for (overlap.h)
typedef overlap::Bytes Bytes;
Bytes bytes_of(const hum_decay_attn_args* p, const hum_rows& r, int heads, int d, int size) {
    return Bytes(r.ptr, (int64_t)d * size).by(p->lanes, r.lane * size).by(p->steps, r.step * size).by(heads, r.head * size);
}
Bytes bytes_of(const hum_decay_attn_args* p, const float* state) {
    return Bytes(state, 4ll * p->lanes * p->heads * p->dk * p->dv);
}
Bytes bytes_of_reset(const hum_decay_attn_args* p) { return Bytes(p->reset, 1).by(p->lanes, p->reset_lane).by(p->steps, p->reset_step); }
Bytes bytes_of_decay(const hum_decay_attn_args* p) { return Bytes(p->log_decay, 4ll * p->heads); }
Bytes bytes_of_lengths(const hum_decay_attn_args* p) { return Bytes(p->lengths, 4ll * p->lanes); }
// a call's state_in, out of the question where state_out is the same
Bytes bytes_of_entering(const hum_decay_attn_args* p) { return p->state_in == p->state_out ? Bytes() : bytes_of(p, p->state_in); }

int in_32(int d) { return d <= 32 ? 1 : d <= 64 ? 2 : 4; }
template <int ST, int K, int W, int J, int HEADS, Mode MODE, bool OUTS>
void launch_walk_j(const WalkArgs& a, hipStream_t s) {
    const long n = (long)a.lanes * a.heads / HEADS * a.segs;
    const dim3 grid((unsigned)((n + XCDS * NEAR - 1) / (XCDS * NEAR) * (XCDS * NEAR) * a.nroles));
    hipLaunchKernelGGL((walk_kernel<ST, K, W, J, HEADS, MODE, OUTS>), grid, dim3(64 * W * HEADS), 0, s, a);
}
// W waves of 32 of z's channels, or 2 W of 16: half of a wave's part of a chunk, while a head's rows are read from LDS twice
// as often.  Thin slices are faster while a wave of 32 channels has a SIMD of its own (thin: bf16, 4 heads x 64 x 64, 200 steps,
// 64 lanes: 21.2 us with wide slices, 18.3; 128 lanes 26.4 and 21.6), wide ones from there on but for some forwards (512 lanes
// 65.5 and 62.4, gradient 136 and 149; 128 channels 163 and 195; 4096 time-major lanes x 32 steps 153 and 192, gradient 300
// and 392).  Thin ones always for types of several parts (but float16 of more than 64 channels: gradient of 512 lanes x 100
// steps x 128 333 and 447) and for unaligned rows of up to 64 channels or of two parts: as measured when wide slices were
// built for them too, float32 4 x 64 x 64, 512 lanes x 200 steps 146 and 125 us, float16 1024 lanes x 100 steps x 127 609
// and 428, bf16 63 channels 121 and 116, gradient 272 and 257.
// Rows of more than 64 channels are work for four waves to load and to form P of, also where z has fewer channels than they
// could hold (float32, 128 x 32 channels, 64 lanes x 100 steps: 28.9 us with two waves, 24.8 with four); with wide slices,
// for many walks, z of up to 32 channels still has one wave, with the registers of a SIMD to itself.
template <int ST, int K, int W, bool OUTS>
void launch_walk_o(const WalkArgs& a, Mode mode, bool together, bool thin, hipStream_t s) {
    constexpr int THIN = K > 2 && W == 1 ? 4 : 2 * W;
    if (mode == BUFFER) {
        if constexpr (ST == HUM_BF16 || (ST == HUM_F16 && K > 2))
            if (!thin) {
                // 4 waves a workgroup from as many heads as that takes, where keys and values are equally wide
                constexpr int H = ST != HUM_BF16 || K != W ? 1 : 4 / W;
                if (together && a.heads % H == 0) return launch_walk_j<ST, K, W, 2, H, BUFFER, OUTS>(a, s);
                return launch_walk_j<ST, K, W, 2, 1, BUFFER, OUTS>(a, s);
            }
        launch_walk_j<ST, K, THIN, 1, 1, BUFFER, OUTS>(a, s);
    } else if (mode == WIDE) {
        if constexpr (ST == HUM_BF16 && K > 2 && W > 2)
            if (!thin) return launch_walk_j<ST, K, W, 2, 1, WIDE, OUTS>(a, s);
        launch_walk_j<ST, K, THIN, 1, 1, WIDE, OUTS>(a, s);
    } else if constexpr (K == W) {
        launch_walk_j<ST, K, THIN, 1, 1, ANY, OUTS>(a, s);
    }
}
template <int ST, int K, int W>
void launch_walk_w(const WalkArgs& a, Mode mode, bool together, bool thin, hipStream_t s) {
    if (a.r[0].x.p) launch_walk_o<ST, K, W, true>(a, mode, together, thin, s);
    else launch_walk_o<ST, K, W, false>(a, mode, together, thin, s);
}
template <int ST, int K>
void launch_walk_k(const WalkArgs& a, int w, Mode mode, bool together, bool thin, hipStream_t s) {
    if (w == 1) launch_walk_w<ST, K, 1>(a, mode, together, thin, s);
    else if (w == 2) launch_walk_w<ST, K, 2>(a, mode, together, thin, s);
    else launch_walk_w<ST, K, 4>(a, mode, together, thin, s);
}
template <int ST>
void launch_walk_t(const WalkArgs& a, hipStream_t s) {
    // together: four heads of a step are neighbours and the steps so far apart that a chunk's 32 rows lie in as many pages
    // (gradient of 4096 x 32 steps, time-major 2 MB apart: 333 us with single heads, 300 us; lane-major 259 and 272 us)
    bool buffers = !a.reset || (a.reset_step >= 0 && a.reset_step < (1l << 25)), wide = true, together = true;
    auto near = [](const Rows& m, int d) { return m.near && d * Num<ST>::SIZE >= 16; };
    auto within = [](const Rows& m, int d) { return m.head >= 0 && 3 * m.head + d <= m.step && m.step * Num<ST>::SIZE >= 1 << 16; };
    for (int i = 0; i < a.nroles; i++) {
        const Role& r = a.r[i];
        buffers = buffers && (!r.x.p || r.x.vec) && r.y.vec && r.z.vec && (!r.out.p || r.out.vec) && r.s_vec;
        wide = wide && (!r.x.p || near(r.x, r.dy)) && near(r.y, r.dy) && near(r.z, r.dz);
        together = together && (!r.x.p || within(r.x, r.dy)) && within(r.y, r.dy) && within(r.z, r.dz) && (!r.out.p || within(r.out, r.dz));
    }
    int k = in_32(a.r[0].dy), w = in_32(a.r[0].dz);
    const Mode mode = buffers ? BUFFER : wide ? WIDE : ANY;
    if (mode == ANY) k = w = k > w ? k : w;   // (that is built for squares only)
    const bool thin = (long)a.lanes * a.heads * a.segs * a.nroles * w <= 1024;
    if (k == 1) launch_walk_k<ST, 1>(a, w, mode, together, thin, s);
    else if (k == 2) launch_walk_k<ST, 2>(a, w, mode, together, thin, s);
    else launch_walk_k<ST, 4>(a, w, mode, together, thin, s);
}

// Few lanes and many steps: the walks are cut into segments that run side by side, each from the state that a first pass
// over the segments before it and a scan have left for it (segments without outputs: half the work of a walk).  Longer
// walks have longer segments (each has a state in memory and a turn in the scan) and more of them side by side; walks
// that would be cut into few, or are short, do not gain what the first pass and two launches cost.  The numbers are fitted to
// measurements, there is no model behind them, and they count a.steps, not the lanes' lengths.  Averages over types, widths
// of 32 to 128 and both directions, against the best cut of each case:
//     12 to 24 chunks,  8 waves: uncut 2.34, segments of 1 chunk 1.00, of 4 1.67;  256 waves: uncut 1.02, up to 2048 waves 1.29
//     32 chunks, 256 waves: uncut 1.09, 2048 waves 1.11;  63 chunks, 256 waves: uncut 1.25, 2048 1.09, 4096 1.06
//     125 chunks, 512 waves: uncut 1.06, 4096 1.02;  250 chunks, 16 waves: segments of 1 chunk 1.13, 2 1.10, 3 1.00, 4 1.09
struct Cut { int segs, steps; };
Cut cut_of(const hum_decay_attn_args* p, int walks) {   // of a (lane, head)
    // in waves of 32 x 32 channels; uneven widths (10 lanes x 7 heads x 907 steps of 117 and 22 channels, float16 gradient:
    // 206 us uncut, 154 cut) take the mean of theirs
    const double waves = (double)p->lanes * p->heads * walks * std::sqrt((double)(in_32(p->dk) * in_32(p->dv)));
    const int chunks = (p->steps + CH - 1) / CH, least = chunks < 32 ? 1 : chunks < 128 ? 2 : 3;
    const int most = chunks < 48 ? 2048 : 4096;
    const bool parts = p->type != HUM_BF16;   // chunks take longer: 29 of them are cut into 5 segments too
    if (waves == 0 || chunks < (parts ? 8 : 12) || waves * (chunks >= 96 ? 4 : parts && chunks >= 20 && chunks < 48 ? 4.5 : 8) > most)
        return {1, p->steps};
    long segs = (long)(most / waves);
    if (segs > chunks / least) segs = chunks / least;
    const int per = (int)((chunks + segs - 1) / segs);
    return {(chunks + per - 1) / per, per * CH};
}

// roles of equal widths share a launch: workgroups that read the same rows run at about the same time
void launch_roles(const hum_decay_attn_args* p, const Role* r, int n, Cut c, bool last_only, hipStream_t s) {
    WalkArgs a = {};
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
    bool done[3] = {};
    for (int i = 0; i < n; i++) {
        if (done[i]) continue;
        a.nroles = 0;
        for (int j = i; j < n; j++)
            if (!done[j] && in_32(r[j].dy) == in_32(r[i].dy) && in_32(r[j].dz) == in_32(r[i].dz)) {
                done[j] = true;
                a.r[a.nroles++] = r[j];
            }
        if (p->type == HUM_BF16) launch_walk_t<HUM_BF16>(a, s);
        else if (p->type == HUM_F16) launch_walk_t<HUM_F16>(a, s);
        else launch_walk_t<HUM_F32>(a, s);
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
// fills the scratch of each walk (n of them) with its segments' entering states; a walk is a role whose y side is the keys'
void run_segments(const hum_decay_attn_args* p, Role* walk, float* const* scratch, int n, Cut c, hipStream_t s) {
    const long units = (long)p->lanes * p->heads, size = (long)p->dk * p->dv;
    ScanArgs a = {};
    a.segs = c.segs;
    a.size = (int)size;
    a.units = units;
    for (int i = 0; i < n; i++) {
        Role& w = walk[i];
        float* through = (float*)((char*)scratch[i] + round16(4 * units * c.segs * size));
        a.w[i].in = w.state_in;
        a.w[i].seg = scratch[i];
        a.w[i].through = through;
        w.x = w.out = Rows{};
        w.x.shared = w.out.shared = 1;
        w.state_in = nullptr;
        w.state_out = scratch[i];
        w.out_unit = size * c.segs;
        w.out_seg = size;
        w.through = through;
        w.s_vec = p->dk % 4 == 0;
    }
    launch_roles(p, walk, n, c, false, s);
    hipLaunchKernelGGL(scan_kernel, dim3((unsigned)((units * size + 255) / 256), n), dim3(256), 0, s, a);
}
void enter_segments(Role& r, const float* scratch, const hum_decay_attn_args* p, Cut c) {
    r.state_in = scratch;
    r.in_unit = (long)p->dk * p->dv * c.segs;
    r.in_seg = (long)p->dk * p->dv;
}
Cut forward_cut(const hum_decay_attn_args* p) { return cut_of(p, 1); }
Cut backward_cut(const hum_decay_attn_args* p) { return cut_of(p, 3); }

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
    const int size = elem_size(p->type), group = p->heads / p->kv_heads;
    const Bytes writes[] = {bytes_of(p, *out, p->heads, p->dv, size), bytes_of(p, p->state_out), Bytes(workspace, need)};
    const Bytes reads[] = {bytes_of(p, p->q, p->heads, p->dk, size), bytes_of(p, p->k, p->kv_heads, p->dk, size),
                           bytes_of(p, p->v, p->kv_heads, p->dv, size), bytes_of_entering(p), bytes_of_decay(p), bytes_of_reset(p),
                           bytes_of_lengths(p)};
    if (overlap::clash(writes, reads))
        return derr(HUM_ERR_ARG, fn, "out, state_out and the workspace must overlap neither each other nor an input (state_out may be state_in)");
    const OnDevice dev(p->device);
    if (!dev.ok) return derr(HUM_ERR_HIP, fn, "hipSetDevice");
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
        Role w = r;
        float* const at = (float*)workspace;
        run_segments(p, &w, &at, 1, c, (hipStream_t)stream);
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
    if (!p->lanes) return HUM_OK;
    const Bytes writes[] = {bytes_of(p, gq, p->heads, p->dk, size), bytes_of(p, gk, p->kv_heads, p->dk, size),
                            bytes_of(p, gv, p->kv_heads, p->dv, size), bytes_of(p, d_state_in), Bytes(workspace, need)};
    const Bytes reads[] = {bytes_of(p, p->q, p->heads, p->dk, size), bytes_of(p, p->k, p->kv_heads, p->dk, size),
                           bytes_of(p, p->v, p->kv_heads, p->dv, size), bytes_of(p, *d_out, p->heads, p->dv, size),
                           bytes_of(p, p->state_in), bytes_of(p, d_state_out), bytes_of_decay(p), bytes_of_reset(p),
                           bytes_of_lengths(p)};
    if (overlap::clash(writes, reads))
        return derr(HUM_ERR_ARG, fn, "gradients and the workspace must overlap neither each other nor an input");
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
        Role w[2];
        float* at[2];
        int m = 0;
        if (gq.ptr) {
            Role& x = w[m] = Role{};
            at[m++] = seg_s;
            x.y = k; x.z = v;
            x.dy = p->dk; x.dz = p->dv;
            x.s_add = 1.f;
            role_state(x, p->state_in, nullptr, p, true);
        }
        if (gk.ptr || gv.ptr || d_state_in) {
            Role& x = w[m] = Role{};
            at[m++] = seg_r;
            x.y = q; x.z = g;
            x.dy = p->dk; x.dz = p->dv;
            x.rev = 1;
            x.s_add = p->scale;
            role_state(x, d_state_out, nullptr, p, true);
        }
        if (m) run_segments(p, w, at, m, c, s);
        for (int i = 0; i < n; i++) enter_segments(r[i], r[i].rev ? seg_r : seg_s, p, c);
    }
    launch_roles(p, r, n, c, true, s);
    if (group > 1 && p->steps && (gk.ptr || gv.ptr)) {
        ShareArgs a = {};
        a.rows = (long)p->lanes * p->steps;
        a.steps = p->steps;
        a.kv = p->kv_heads;
        a.group = group;
        a.x[0] = {part_k, rows_of(gk, 1, size, p->dk), p->dk};
        a.x[1] = {part_v, rows_of(gv, 1, size, p->dv), p->dv};
        const long blocks = (a.rows * a.kv * (p->dk > p->dv ? p->dk : p->dv) + 255) / 256;
        const dim3 grid((unsigned)(blocks < (1 << 16) ? blocks : (1 << 16)), 2);
        if (p->type == HUM_F32) hipLaunchKernelGGL(share_kernel<HUM_F32>, grid, dim3(256), 0, s, a);
        else if (p->type == HUM_BF16) hipLaunchKernelGGL(share_kernel<HUM_BF16>, grid, dim3(256), 0, s, a);
        else hipLaunchKernelGGL(share_kernel<HUM_F16>, grid, dim3(256), 0, s, a);
    }
    return launched(fn);
}

}  // extern "C"

namespace {
template <int ST>
void launch_step(const StepArgs& a, int lpr, dim3 grid, hipStream_t s) {
    switch (lpr) {
        case 1: hipLaunchKernelGGL((step_kernel<ST, 1>), grid, dim3(256), 0, s, a); break;
        case 2: hipLaunchKernelGGL((step_kernel<ST, 2>), grid, dim3(256), 0, s, a); break;
        case 4: hipLaunchKernelGGL((step_kernel<ST, 4>), grid, dim3(256), 0, s, a); break;
        case 8: hipLaunchKernelGGL((step_kernel<ST, 8>), grid, dim3(256), 0, s, a); break;
        case 16: hipLaunchKernelGGL((step_kernel<ST, 16>), grid, dim3(256), 0, s, a); break;
        default: hipLaunchKernelGGL((step_kernel<ST, 32>), grid, dim3(256), 0, s, a); break;
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
    const int size = elem_size(p->type), group = p->heads / p->kv_heads;
    // (a head's workgroups and waves read all of q and k, and store their rows of out and of the state at once)
    const Bytes writes[] = {bytes_of(p, *out, p->heads, p->dv, size), bytes_of(p, p->state_out)};
    const Bytes reads[] = {bytes_of(p, p->q, p->heads, p->dk, size), bytes_of(p, p->k, p->kv_heads, p->dk, size),
                           bytes_of(p, p->v, p->kv_heads, p->dv, size), bytes_of_entering(p), bytes_of_decay(p), bytes_of_reset(p),
                           Bytes(active, p->lanes)};
    if (overlap::clash(writes, reads))
        return derr(HUM_ERR_ARG, fn, "out and state_out must overlap neither each other nor an input (state_out may be state_in)");
    const OnDevice dev(p->device);
    if (!dev.ok) return derr(HUM_ERR_HIP, fn, "hipSetDevice");
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
    int lpr = 1;
    while (4 * lpr < p->dk) lpr *= 2;
    const int rows = 4 * 4 * (64 / lpr);
    a.blocks = (p->dv + rows - 1) / rows;
    const dim3 grid((unsigned)(p->lanes * p->heads * a.blocks));
    if (p->type == HUM_BF16) launch_step<HUM_BF16>(a, lpr, grid, (hipStream_t)stream);
    else if (p->type == HUM_F16) launch_step<HUM_F16>(a, lpr, grid, (hipStream_t)stream);
    else launch_step<HUM_F32>(a, lpr, grid, (hipStream_t)stream);
    return launched(fn);
}
