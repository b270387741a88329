// Tiled matrix products on the matrix cores, shared by the linear layers and
// Muon: D(i, j) = sum over k of A(i, k) B(j, k), float sums.
//
// Each operand is read in one of two forms: K-contiguous (element (r, k) at
// p + r stride + k) or R-contiguous (p + k stride + r). A workgroup of
// WI x WJ waves makes a tile of BI x BJ outputs, a wave TI x TJ squares of
// 16 x 16, in steps of 128 bytes of k (64 halves, 32 floats); Muon's R-contiguous side
// takes 64.
//
// Operand tiles go from memory to LDS without passing registers: lane l of a
// wave's load writes the 16 bytes at its LDS base + 16 l, from any byte
// address and zeros when the address is past the buffer's end, which is how
// edges are filled. A ring of stages: the loads of the next steps are in
// flight while a step is multiplied; one barrier a step. A step's fragments
// are read into registers while the step before it is multiplied: read at its
// own start, the matrix cores waited for LDS (16384 x 2048 -> 1024 gradients:
// 75 us). LDS is read without conflicts
// because the 16-byte chunks of a row are permuted by the row's number: the
// lanes choose which chunk they fetch.
#pragma once

#include "common.h"
#include "network.h"

namespace tgs {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

template <class T>
struct Frag;
template <>
struct Frag<_Float16> {
    typedef _Float16 type __attribute__((ext_vector_type(8)));
};
template <>
struct Frag<__bf16> {
    typedef __bf16 type __attribute__((ext_vector_type(8)));
};
// A float is held as three bfloat16, high + middle + low: 24 bits in all, each
// the nearest to what the ones before leave. For infinities, NaN and floats of
// 2^128 (1 - 2^-9) and more high is not finite, and so is every sum that they
// enter, whatever it should be (inf - inf, 0 inf): form_again mends those.
template <>
struct Frag<float> {
    typedef __bf16 plane __attribute__((ext_vector_type(8)));
    struct type {
        plane high, middle, low;
    };
};

// Two floats to their nearest bfloat16 (in one word: one conversion makes
// both), and what is left of them.
__device__ __forceinline__ uint32_t take_bf16(float& x, float& y) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const uint32_t u = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{x, y}), bf16x2));
    x -= __builtin_bit_cast(float, u << 16);
    y -= __builtin_bit_cast(float, u & 0xffff0000u);
    return u;
}

__device__ __forceinline__ Frag<float>::type split3(const float (&v)[8]) {
    typedef uint32_t words __attribute__((ext_vector_type(4)));
    words p[3];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float x = v[2 * e], y = v[2 * e + 1];
#pragma unroll
        for (int q = 0; q < 3; ++q) p[q][e] = take_bf16(x, y);
    }
    return {__builtin_bit_cast(Frag<float>::plane, p[0]), __builtin_bit_cast(Frag<float>::plane, p[1]),
            __builtin_bit_cast(Frag<float>::plane, p[2])};
}

// Products of a 16 x 16 square over 32 of k. Row 4 (lane / 16) + r of the
// square is in register r, column lane % 16. Floats: six of the nine plane
// products (the others are below 2^-25 of the whole), 96 cycles where the
// matrix cores' float instructions take 256.
__device__ __forceinline__ f32x4 multiply(Frag<_Float16>::type a, Frag<_Float16>::type b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 multiply(Frag<__bf16>::type a, Frag<__bf16>::type b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 multiply(const Frag<float>::type& a, const Frag<float>::type& b, f32x4 c) {
    c = multiply(a.low, b.high, c);
    c = multiply(a.high, b.low, c);
    c = multiply(a.middle, b.middle, c);
    c = multiply(a.middle, b.high, c);
    c = multiply(a.high, b.middle, c);
    return multiply(a.high, b.high, c);
}

// Float outputs that came out infinite or NaN, formed again from the operands by
// the matrix cores' float instructions, so that they are what float products
// and sums give; the others keep their bits. fa(u, a, k) and fb(v, a, k) are
// rows 16 u + a of A and 16 v + a of B at k, which runs from k0 to below k1;
// exists(u, v, r) tells the lane whether its register r of a square is an
// output at all. A wave looks at its own squares, one multiply-add a register
// (16384 x 1024 -> 2048 floats 345 us without it and 348 with it, 1e6 x 128 ->
// 128 274 and 281); where it finds something it takes several times the
// products' time.
template <int TI, int TJ, class FA, class FB, class Exists>
__device__ __forceinline__ void form_again(f32x4 (&acc)[TI][TJ], int64_t k0, int64_t k1, FA fa, FB fb, Exists exists) {
    f32x4 none = {0.0f, 0.0f, 0.0f, 0.0f};   // 0 where all are finite
#pragma unroll
    for (int u = 0; u < TI; ++u)
#pragma unroll
        for (int v = 0; v < TJ; ++v)
#pragma unroll
            for (int r = 0; r < 4; ++r) none[r] = fmaf(acc[u][v][r], 0.0f, none[r]);
    if (ballot((none[0] + none[1]) + (none[2] + none[3]) != 0.0f) == 0) return;
    const int a = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3;
#pragma unroll
    for (int u = 0; u < TI; ++u) {
        bool ends = false;
#pragma unroll
        for (int v = 0; v < TJ; ++v)
#pragma unroll
            for (int r = 0; r < 4; ++r) ends |= !__builtin_isfinite(acc[u][v][r]) && exists(u, v, r);
        if (ballot(ends) == 0) continue;
        f32x4 sum[TJ];
#pragma unroll
        for (int v = 0; v < TJ; ++v) sum[v] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
        for (int64_t from = k0; from < k1; from += 4) {
            const int64_t k = from + g;
            const float x = k < k1 ? fa(u, a, k) : 0.0f;
#pragma unroll
            for (int v = 0; v < TJ; ++v)
                sum[v] = __builtin_amdgcn_mfma_f32_16x16x4f32(x, k < k1 ? fb(v, a, k) : 0.0f, sum[v], 0, 0, 0);
        }
#pragma unroll
        for (int v = 0; v < TJ; ++v)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[u][v][r] = __builtin_isfinite(acc[u][v][r]) ? acc[u][v][r] : sum[v][r];
    }
}

// An operand of a launch. K-contiguous: `rows` of `cols` = k elements;
// R-contiguous: `rows` = k of `cols` elements.
struct TileOperand {
    const void* p;
    int64_t rows, cols, stride;
};

constexpr uint32_t kPastEnd = 0xffffff00u;   // an offset past every buffer's end

typedef __attribute__((address_space(3))) unsigned char lds_byte;

__device__ __forceinline__ uint32_t lds_address(void* p) { return (uint32_t)(uintptr_t)(lds_byte*)p; }

// 16 bytes a lane from buffer + offset to LDS at base + 16 lane. The base goes
// through m0, a register that asm cannot declare as changed: it is put back.
__device__ __forceinline__ void load_to_lds(uint32_t base, uint32_t offset, i32x4 buffer) {
    uint32_t held;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, 0 offen lds\n\t"
                 "s_mov_b32 m0, %0"
                 : "=&s"(held)
                 : "s"(__builtin_amdgcn_readfirstlane(base)), "v"(offset), "s"(buffer)
                 : "memory");
}

__device__ __forceinline__ i32x4 buffer_of(const void* p, int64_t bytes) {
    const uint64_t a = (uint64_t)p;
    const uint32_t n = bytes <= 0 ? 0u : bytes < (int64_t)kPastEnd ? (uint32_t)bytes : kPastEnd;
    i32x4 r;
    r[0] = __builtin_amdgcn_readfirstlane((int)(uint32_t)a);
    r[1] = __builtin_amdgcn_readfirstlane((int)((uint32_t)(a >> 32) & 0xffffu));
    r[2] = __builtin_amdgcn_readfirstlane((int)n);
    r[3] = 0x00020000;
    return r;
}

// The same for the compiler's own buffer loads and stores. A load past the end
// gives zeros and a store there is dropped, so that edges need no branches.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t resource_of(const void* p, int64_t bytes) {
    const uint32_t n = bytes <= 0 ? 0u : bytes < (int64_t)kPastEnd ? (uint32_t)bytes : kPastEnd;
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)n, 0x00020000);
}
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// One operand's side of a tile: R rows (i or j), loaded by WAVES waves, STEP
// bytes of k a step.
template <class T, int R, int WAVES, bool RC, int STEP = 128>
struct TileSide {
    static constexpr int V = 16 / (int)sizeof(T);             // elements of a chunk
    static constexpr int kDepth = STEP / (int)sizeof(T);   // k of a step
    static constexpr int kBytes = R * STEP;
    static constexpr int kLoads = kBytes / 1024 / WAVES;      // per wave and step
    static_assert(STEP == 128 || STEP == 64, "");
    static_assert(kLoads >= 1 && kLoads * 1024 * WAVES == kBytes, "a whole number of loads a wave");
    static constexpr int kRowBytes = RC ? R * (int)sizeof(T) : STEP;   // of an LDS row
    static constexpr int kRowChunks = kRowBytes / 16;

    // The chunk that stands in place of chunk c of LDS row r, and back.
    // K-contiguous: lanes 0..15 read rows r .. r + 15 at one chunk, so chunks
    // are turned by the row (by every fourth where four rows fill the banks).
    // R-contiguous: a read takes 4 (halves: 8) rows at one run of 16 elements,
    // so the runs are turned by what tells the rows (8 g + q, floats: 8 g + e at
    // one e) apart; rows of 128 bytes already alternate between the banks' halves.
    static __device__ __forceinline__ int turn(int r) {
        if constexpr (!RC) return STEP == 128 ? r & 7 : (r >> 2) & 3;
        if constexpr (sizeof(T) == 4) return ((r >> 3) & 3) << 2;
        if constexpr (kRowBytes == 128) return (((r >> 1) & 1) | (((r >> 3) & 1) << 1)) << 1;
        return ((r & 3) | (((r >> 3) & 1) << 2)) << 1;
    }

    const unsigned char* base;   // of the tile's first step
    int64_t end;                 // bytes of the buffer from base
    int64_t step_bytes;
    uint32_t offset[kLoads];
    int row_bytes;               // R-contiguous: bytes of a row within the tile that hold elements

    // Tile of rows r0 .. and steps from k0 on.
    __device__ __forceinline__ void begin(const TileOperand& o, int64_t r0, int64_t k0, int wave, int lane) {
        const int64_t pitch = o.stride * (int64_t)sizeof(T);
        const int64_t whole = (o.rows - 1) * pitch + o.cols * (int64_t)sizeof(T);
        const int64_t at = RC ? k0 * pitch + r0 * (int64_t)sizeof(T) : r0 * pitch + k0 * (int64_t)sizeof(T);
        base = (const unsigned char*)o.p + at;
        end = whole - at;
        step_bytes = RC ? kDepth * pitch : STEP;
        const int64_t left = RC ? o.cols - r0 : o.rows - r0;   // rows of the tile that exist
        row_bytes = (int)(left < R ? left : R) * (int)sizeof(T);
#pragma unroll
        for (int n = 0; n < kLoads; ++n) {
            const int slot = (n * WAVES + wave) * 64 + lane;
            const int r = slot / kRowChunks, c = (slot % kRowChunks) ^ turn(r);
            const bool exists = RC ? c * 16 < row_bytes : r < left;
            offset[n] = exists ? (uint32_t)(r * pitch + c * 16) : kPastEnd;
        }
    }

    // Starts the loads of a step into `lds`; `left` of k remain from its
    // start. Chunks past k are zeros. The chunk that holds the last elements
    // of k (K-contiguous), or of the matrix (R-contiguous: a chunk past a
    // row's end is filled from the next row, into outputs that do not exist),
    // is gathered element by element.
    __device__ __forceinline__ void load(unsigned char* lds, int64_t left, int wave, int lane) {
        const i32x4 buffer = buffer_of(base, end);
        const uint32_t to = lds_address(lds);
        const bool inside = RC ? left > kDepth || (left == kDepth && row_bytes % 16 == 0)
                               : left >= kDepth;
        if (inside) {
#pragma unroll
            for (int n = 0; n < kLoads; ++n) load_to_lds(to + (n * WAVES + wave) * 1024, offset[n], buffer);
        } else {
#pragma unroll
            for (int n = 0; n < kLoads; ++n) {
                const int slot = (n * WAVES + wave) * 64 + lane;
                const int r = slot / kRowChunks, c = (slot % kRowChunks) ^ turn(r);
                // elements of the chunk that exist: all, none or some
                int some;
                if constexpr (RC) some = r + 1 < left ? V : r < left ? (row_bytes - c * 16) / (int)sizeof(T) : 0;
                else some = (int)left - c * V;
                const bool exists = offset[n] != kPastEnd && some > 0;
                if (some >= V || !exists) {
                    load_to_lds(to + (n * WAVES + wave) * 1024, exists ? offset[n] : kPastEnd, buffer);
                } else {
                    const T* p = (const T*)(base + offset[n]);
                    T* q = (T*)(lds + slot * 16);
#pragma unroll
                    for (int e = 0; e < V; ++e) q[e] = e < some ? p[e] : (T)0.0f;
                }
            }
        }
        base += step_bytes;
        end -= step_bytes;
    }

    static constexpr int kSubs = kDepth / 32;   // multiply()s of a step

    // The fragment of rows r0 .. r0 + 15 (r0 a multiple of 16) at part s of a step.
    static __device__ __forceinline__ typename Frag<T>::type fragment(const unsigned char* lds, int r0, int s, int lane) {
        const int a = lane & 15, g = lane >> 4;
        if constexpr (sizeof(T) == 4) {
            float x[8];
            if constexpr (!RC) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const f32x4 v = *(const f32x4*)(lds + (r0 + a) * STEP + (((2 * g + h) ^ turn(a)) << 4));
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[4 * h + e] = v[e];
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int k = 8 * g + e;
                    x[e] = *(const float*)(lds + k * kRowBytes + (((r0 >> 4) ^ (turn(k) >> 2)) << 6) + a * 4);
                }
            }
            return split3(x);
        } else if constexpr (!RC) {
            return *(const typename Frag<T>::type*)(lds + (r0 + a) * STEP + (((4 * s + g) ^ turn(a)) << 4));
        } else {
            // the transposing read: lanes 4 q .. 4 q + 3 of 16 name row q's
            // four runs of 8 bytes, and lane l receives column l of the rows
            const int q = a >> 2, k = 32 * s + 8 * g + q;
            const int at = ((r0 >> 4) ^ (turn(8 * g + q) >> 1)) * 32 + (a & 3) * 8;
            typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
            union {
                i16x4 half[2];
                typename Frag<T>::type whole;
            } u;
            u.half[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(lds_byte*)(lds + k * kRowBytes + at));
            const int at4 = ((r0 >> 4) ^ (turn(8 * g + q + 4) >> 1)) * 32 + (a & 3) * 8;
            u.half[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(lds_byte*)(lds + (k + 4) * kRowBytes + at4));
            return u.whole;
        }
    }
};

// Waits until at most n (0 or 1) groups of L of the wave's loads are in flight
// and its LDS accesses are done, then for the workgroup.
template <int L>
__device__ __forceinline__ void wait_for_stage(int n) {
    static_assert(L < 64, "what the counter holds");
    if (n > 0) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(L) : "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Rows (4 registers) of squares t and t + 1 of a lane, exchanged between the
// 16-lane rows so that the lane holds 8 neighbouring outputs: squares t, t + 1
// at i0 + 8 (lane / 32) + 16 ((lane / 16) % 2) .. + 7.
__device__ __forceinline__ void neighbours(const f32x4& a, const f32x4& b, float (&v)[8]) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        v[r] = a[r];
        v[4 + r] = b[r];
        swap16(v[r], v[4 + r]);
    }
}
__device__ __forceinline__ int neighbours_at(int lane) { return 8 * (lane >> 5) + 16 * ((lane >> 4) & 1); }

// The tile at (i0, j0) over k in [k0, k1): acc[ti][tj] of each wave. `lds`
// holds the stages. k0 is a multiple of a step.
template <class T, int WI, int WJ, int TI, int TJ, bool A_RC, bool B_RC, int STEP, int STAGES>
struct Tile {
    static constexpr int kWaves = WI * WJ, kThreads = 64 * kWaves;
    static constexpr int BI = WI * TI * 16, BJ = WJ * TJ * 16;
    using A = TileSide<T, BI, kWaves, A_RC, STEP>;
    using B = TileSide<T, BJ, kWaves, B_RC, STEP>;
    static constexpr int kStage = A::kBytes + B::kBytes;
    static constexpr int kLds = STAGES * kStage;
    static constexpr int kLoads = A::kLoads + B::kLoads;   // at least these many a wave and stage (gathers add some)
    static_assert(STAGES == 2, "what wait_for_stage waits for");

    static __device__ __forceinline__ void run(unsigned char* lds, const TileOperand& a, const TileOperand& b, int64_t i0,
                                               int64_t j0, int64_t k0, int64_t k1, f32x4 (&acc)[TI][TJ]) {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int wi = wave / WJ, wj = wave % WJ;
        A sa;
        B sb;
        sa.begin(a, i0, k0, wave, lane);
        sb.begin(b, j0, k0, wave, lane);
#pragma unroll
        for (int u = 0; u < TI; ++u)
#pragma unroll
            for (int v = 0; v < TJ; ++v) acc[u][v] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        const int steps = (int)((k1 - k0 + A::kDepth - 1) / A::kDepth);
        if (steps <= 0) return;
        int64_t left = k1 - k0;   // of k from the next load on
        unsigned char* fill = lds;
        const auto load = [&] {
            sa.load(fill, left, wave, lane);
            sb.load(fill + A::kBytes, left, wave, lane);
            left -= A::kDepth;
            fill = fill + kStage < lds + kLds ? fill + kStage : lds;
        };
        const unsigned char* from = lds;   // the stage of the next read
        if constexpr (sizeof(T) == 4) {
            static_assert(A::kSubs == 1, "");
            load();
            for (int t = 0; t < steps; ++t) {
                wait_for_stage<kLoads>(0);
                if (t + 1 < steps) load();
                typename Frag<T>::type fb[TJ];
#pragma unroll
                for (int v = 0; v < TJ; ++v) fb[v] = B::fragment(from + A::kBytes, (wj * TJ + v) * 16, 0, lane);
#pragma unroll
                for (int u = 0; u < TI; ++u) {   // twelve registers a fragment: one of A at a time
                    const auto fa = A::fragment(from, (wi * TI + u) * 16, 0, lane);
#pragma unroll
                    for (int v = 0; v < TJ; ++v) acc[u][v] = multiply(fa, fb[v], acc[u][v]);
                }
                from = from + kStage < lds + kLds ? from + kStage : lds;
            }
            const int64_t ni = A_RC ? a.cols : a.rows, nj = B_RC ? b.cols : b.rows;
            const int64_t iw = i0 + wi * TI * 16, jw = j0 + wj * TJ * 16;
            // outputs that do not exist hold what follows a row in memory
            form_again(
                acc, k0, k1,
                [&](int u, int row, int64_t k) {
                    const int64_t i = iw + 16 * u + row;
                    return i < ni ? ((const T*)a.p)[A_RC ? k * a.stride + i : i * a.stride + k] : 0.0f;
                },
                [&](int v, int row, int64_t k) {
                    const int64_t j = jw + 16 * v + row;
                    return j < nj ? ((const T*)b.p)[B_RC ? k * b.stride + j : j * b.stride + k] : 0.0f;
                },
                [&](int u, int v, int r) { return iw + 16 * u + 4 * (lane >> 4) + r < ni && jw + 16 * v + (lane & 15) < nj; });
        } else {
#pragma unroll
            for (int n = 0; n < STAGES; ++n)
                if (n < steps) load();
            // Two sets of fragments, of a stage's two parts. Each is read while
            // the other is multiplied, so that the reads are done well before
            // the barrier that gives their stage up.
            static_assert(A::kSubs == 2, "");
            typename Frag<T>::type fa[2][TI], fb[2][TJ];
            const auto read = [&](int s) {
#pragma unroll
                for (int v = 0; v < TJ; ++v) fb[s][v] = B::fragment(from + A::kBytes, (wj * TJ + v) * 16, s, lane);
#pragma unroll
                for (int u = 0; u < TI; ++u) fa[s][u] = A::fragment(from, (wi * TI + u) * 16, s, lane);
            };
            const auto multiply_all = [&](int s) {
#pragma unroll
                for (int u = 0; u < TI; ++u)
#pragma unroll
                    for (int v = 0; v < TJ; ++v) acc[u][v] = multiply(fa[s][u], fb[s][v], acc[u][v]);
            };
            wait_for_stage<kLoads>(min(steps - 1, STAGES - 1));
            read(0);
            for (int t = 0; t + 1 < steps; ++t) {
                read(1);
                multiply_all(0);
                // the next stage is there, and every wave has read this one, which the load fills anew
                wait_for_stage<kLoads>(min(steps - 2 - t, STAGES - 2));
                if (t + STAGES < steps) load();
                from = from + kStage < lds + kLds ? from + kStage : lds;
                read(0);
                multiply_all(1);
            }
            read(1);
            multiply_all(0);
            multiply_all(1);
        }
    }
};

// Which tile number n of ni x nj is: runs of `kGroup` j tiles, i outside, so
// that neighbouring numbers cover a block of few operand tiles of each side.
// With the numbers given out by xcd_contiguous_index, that block is what an
// XCD works on and its L2 holds.
__device__ __forceinline__ void tile_of(uint32_t n, uint32_t ni, uint32_t nj, uint32_t& ti, uint32_t& tj) {
    constexpr uint32_t kGroup = 8;
    const uint32_t per = kGroup * ni, group = n / per, in = n % per;
    const uint32_t height = min(kGroup, nj - group * kGroup);
    ti = in / height;
    tj = group * kGroup + in % height;
}

}  // namespace tgs
