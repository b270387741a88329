// What attention's forward and backward share: squares of 32 x 32 on the matrix
// cores, tiles of rows in LDS that are read along and across, and which rows
// of a call a workgroup takes.
//
// A square D(m, n) = sum over k of A(m, k) B(n, k) has column n = lane % 32 and
// rows (r & 3) + 8 (r >> 2) + 4 (lane / 32) in registers r = 0 .. 15. A step
// takes 32 bytes of k of each operand, a chunk of 16 in each half of the lanes.
// Which k a step's places stand for is free as long as both operands agree.
// That is used twice: an operand's own rows are read in chunks of 16 bytes, and a
// square's registers are, once rounded, the B operand of a product over its
// rows: the weights never leave their registers between the two products. Their
// place (half h, element e) then is row 4 h + (e & 3) + 8 (e >> 2) of a step,
// and the A operand is read from LDS in that order.
#pragma once

#include <math.h>

#include "mfma_tile.h"

namespace tgs {

typedef float f32x16 __attribute__((ext_vector_type(16)));

template <class T>
struct Square {   // halves: 16 of k a step
    static constexpr int kDepth = 16;
    using Frag = typename tgs::Frag<T>::type;
    static __device__ __forceinline__ void multiply(const Frag& a, const Frag& b, f32x16& c);
    static __device__ __forceinline__ f32x16 product(const Frag& a, const Frag& b);   // on its own
    // Registers 8 u .. 8 u + 7 of a square, rounded.
    static __device__ __forceinline__ Frag rounded(const f32x16& s, int u) {
        typedef float f32x8 __attribute__((ext_vector_type(8)));
        f32x8 v;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = s[8 * u + e];
        return __builtin_convertvector(v, Frag);
    }
    // What they were rounded by, rounded. INFINITE: there may be infinities, beside which it is nothing.
    template <bool INFINITE>
    static __device__ __forceinline__ Frag rest(const f32x16& s, int u, const Frag& whole) {
        typedef float f32x8 __attribute__((ext_vector_type(8)));
        f32x8 v;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float x = s[8 * u + e] - (float)whole[e];
            v[e] = !INFINITE || fabsf(x) < INFINITY ? x : 0.0f;
        }
        return __builtin_convertvector(v, Frag);
    }
};
template <>
__device__ __forceinline__ void Square<_Float16>::multiply(const Frag& a, const Frag& b, f32x16& c) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x16 Square<_Float16>::product(const Frag& a, const Frag& b) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, f32x16{}, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x16 Square<__bf16>::product(const Frag& a, const Frag& b) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, f32x16{}, 0, 0, 0);
}
template <>
__device__ __forceinline__ void Square<__bf16>::multiply(const Frag& a, const Frag& b, f32x16& c) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
template <>
struct Square<float> {
    static constexpr int kDepth = 8;
    using Frag = f32x4;
    static __device__ __forceinline__ void multiply(const Frag& a, const Frag& b, f32x16& c) {
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x16 product(const Frag& a, const Frag& b) {
        f32x16 c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[0], b[0], f32x16{}, 0, 0, 0);
#pragma unroll
        for (int e = 1; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
        return c;
    }
    static __device__ __forceinline__ Frag rounded(const f32x16& s, int u) {
        return Frag{s[4 * u], s[4 * u + 1], s[4 * u + 2], s[4 * u + 3]};
    }
};

// Row of register r of a square.
__device__ __forceinline__ int square_row(int r, int lane) { return (r & 3) + 8 * (r >> 2) + 4 * (lane >> 5); }

// ROWS rows of one head in LDS, D (a multiple of 32) columns each, the columns
// past the head zeros. The chunks of a row stand turned by its number, so that
// neither sixteen rows' reads of one chunk nor four rows' reads of 64 bytes meet
// on a bank.
template <class T, int D, int ROWS, int WAVES>
struct RowTile {
    static constexpr int V = 16 / (int)sizeof(T);
    static constexpr int kRowBytes = D * (int)sizeof(T);
    static constexpr int kChunks = kRowBytes / 16;
    static constexpr int kBytes = ROWS * kRowBytes;
    static constexpr int kLoads = kBytes / 1024 / WAVES;   // a wave's
    static_assert(kLoads >= 1 && kLoads * 1024 * WAVES == kBytes, "a whole number of loads a wave");
    using S = Square<T>;

    static __device__ __forceinline__ int turn(int r) {
        if constexpr (kRowBytes % 256 == 0) return ((r & 3) << 2) | ((r >> 2) & 3);
        else if constexpr (kRowBytes % 128 == 0) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
        else return (r >> 2) & 3;
    }

    uint32_t offset[kLoads];   // of the thread's chunks from the tile's first row

    // d: the head's columns, pitch: bytes from row to row.
    __device__ __forceinline__ void begin(int64_t pitch, int d, int wave, int lane) {
#pragma unroll
        for (int n = 0; n < kLoads; ++n) {
            const int slot = (n * WAVES + wave) * 64 + lane;
            const int r = slot / kChunks, c = (slot % kChunks) ^ turn(r);
            offset[n] = c * V < d ? (uint32_t)(r * pitch + c * 16) : kPastEnd;
        }
    }

    // Starts the loads of the rows that `exist` has bits for, from `base` on; the
    // others, and the columns past d, are zeros. `end`: bytes from base that may
    // be read. A chunk that the head ends in is gathered element by element.
    __device__ __forceinline__ void load(unsigned char* lds, const unsigned char* base, int64_t end, uint64_t exist, int d,
                                         int wave, int lane) const {
        const i32x4 buffer = buffer_of(base, end);
        const uint32_t to = lds_address(lds);
        constexpr uint64_t kAll = ROWS == 64 ? ~0ull : (1ull << (ROWS & 63)) - 1;
        if (exist == kAll && d % V == 0) {
#pragma unroll
            for (int n = 0; n < kLoads; ++n) load_to_lds(to + (n * WAVES + wave) * 1024, offset[n], buffer);
            return;
        }
#pragma unroll
        for (int n = 0; n < kLoads; ++n) {
            const int slot = (n * WAVES + wave) * 64 + lane;
            const int r = slot / kChunks, c = (slot % kChunks) ^ turn(r);
            const bool exists = offset[n] != kPastEnd && (exist >> r & 1);
            const int some = d - c * V;
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

    // The same of the first `rows` rows (1 or more), the others zeros, or COPIES of the last: where zeros would be NaN
    // beside an infinity of the other operand, a copy only is what that row is. pitch: as in begin. WHOLE: heads of
    // whole chunks.
    template <bool COPIES, bool WHOLE>
    __device__ __forceinline__ void load_first(unsigned char* lds, const unsigned char* base, int64_t end, int64_t rows,
                                               int64_t pitch, int d, int wave, int lane) const {
        const i32x4 buffer = buffer_of(base, end);
        const uint32_t to = lds_address(lds);
        if (rows >= ROWS && (WHOLE || d % V == 0)) {
#pragma unroll
            for (int n = 0; n < kLoads; ++n) load_to_lds(to + (n * WAVES + wave) * 1024, offset[n], buffer);
            return;
        }
        const int last = (int)min(rows, (int64_t)ROWS) - 1;
#pragma unroll
        for (int n = 0; n < kLoads; ++n) {
            const int slot = (n * WAVES + wave) * 64 + lane;
            const int r = slot / kChunks, c = (slot % kChunks) ^ turn(r);
            const int some = d - c * V;
            const bool exists = some > 0 && (COPIES || r <= last);
            const uint32_t at = COPIES ? offset[n] - (uint32_t)max(r - last, 0) * (uint32_t)pitch : offset[n];
            if (WHOLE || some >= V || !exists) {
                load_to_lds(to + (n * WAVES + wave) * 1024, exists ? at : kPastEnd, buffer);
            } else {
                const T* p = (const T*)(base + at);
                T* q = (T*)(lds + slot * 16);
#pragma unroll
                for (int e = 0; e < V; ++e) q[e] = e < some ? p[e] : (T)0.0f;
            }
        }
    }

    // Operand of 32 rows along step s of their columns. lds: the first row, a multiple of 32.
    static __device__ __forceinline__ typename S::Frag along(const unsigned char* lds, int s, int lane) {
        const int r = lane & 31;
        return *(const typename S::Frag*)(lds + r * kRowBytes + (((2 * s + (lane >> 5)) ^ turn(r)) << 4));
    }

    // Operand of columns c0 .. c0 + 31 (a multiple of 32) across the rows
    // r0 .. r0 + kDepth - 1 of the 32 from lds on, in the order of a square's registers.
    static __device__ __forceinline__ typename S::Frag across(const unsigned char* lds, int r0, int c0, int lane) {
        if constexpr (sizeof(T) == 4) {
            typename S::Frag f;
            const int c = c0 + (lane & 31);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = r0 + 4 * (lane >> 5) + e;
                f[e] = *(const float*)(lds + r * kRowBytes + (((c >> 2) ^ turn(r)) << 4) + (c & 3) * 4);
            }
            return f;
        } else {
            // the transposing read: lanes 4 q .. 4 q + 3 of 16 name row q's four runs of 8 bytes, and lane l
            // receives column l of the four rows
            const int a = lane & 15, half = lane >> 5;
            typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
            union {
                i16x4 part[2];
                typename S::Frag whole;
            } u;
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const int r = r0 + 8 * p + 4 * half + (a >> 2);
                const int c = c0 / 8 + 2 * ((lane >> 4) & 1) + ((a & 3) >> 1);
                u.part[p] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (lds_i16x4*)(lds_byte*)(lds + r * kRowBytes + ((c ^ turn(r)) << 4) + (a & 1) * 8));
            }
            return u.whole;
        }
    }

    // Of a 16 x 16 square's product over 32 rows from r0 on: columns c0 .. c0 + 15, and the
    // rows in the order 4 (lane / 16) + (e & 3) + 16 (e >> 2).
    static __device__ __forceinline__ typename S::Frag across16(const unsigned char* lds, int r0, int c0, int lane) {
        static_assert(sizeof(T) == 2, "");
        const int a = lane & 15;
        typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
        union {
            i16x4 part[2];
            typename S::Frag whole;
        } u;
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            const int r = r0 + 16 * p + 4 * (lane >> 4) + (a >> 2);
            const int c = c0 / 8 + ((a & 3) >> 1);
            u.part[p] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (lds_i16x4*)(lds_byte*)(lds + r * kRowBytes + ((c ^ turn(r)) << 4) + (a & 1) * 8));
        }
        return u.whole;
    }
};

// The rows that 32 QB lanes of a wave take, of those that read one head of the
// states in one element of a batch: number i is row i / shared of the element, head
// first + i % shared, so that heads that share lie side by side.
template <int QB>
struct LaneRows {
    int64_t base;      // the first lane's row
    int down[QB];      // the lane's, from there
    int head[QB];
    bool exists[QB];

    __device__ __forceinline__ void begin(int64_t element_row, int64_t i0, int64_t count, int first, int shared, int lane) {
        const int64_t r0 = shared == 1 ? i0 : i0 / shared;
        const uint32_t left = (uint32_t)(i0 - r0 * shared);
        base = element_row + r0;
#pragma unroll
        for (int n = 0; n < QB; ++n) {
            const uint32_t i = 32 * n + (lane & 31);
            exists[n] = i0 + i < count;
            const uint32_t at = left + i;   // below shared + 64
            down[n] = (int)(shared == 1 ? at : at / (uint32_t)shared);
            head[n] = first + (int)(shared == 1 ? 0 : at - (uint32_t)down[n] * (uint32_t)shared);
        }
    }
    __device__ __forceinline__ int64_t row(int n) const { return base + down[n]; }

    // The lanes' chunks of matrix m: chunk 2 s + lane / 32 in f[n][s]. Columns past
    // the head and rows that do not exist are zeros.
    template <class T, int STEPS>
    __device__ __forceinline__ void load(const Mat& m, int d, int lane, typename Square<T>::Frag (&f)[QB][STEPS]) const {
        using F = typename Square<T>::Frag;
        constexpr int V = 16 / (int)sizeof(T);
        const int64_t pitch = m.stride * (int64_t)sizeof(T);
        const unsigned char* from = (const unsigned char*)m.p + base * pitch;
        // whole chunks: all loads on their way at once, without branches
        const auto buffer = resource_of(from, (m.rows - 1 - base) * pitch + m.cols * (int64_t)sizeof(T));
#pragma unroll
        for (int n = 0; n < QB; ++n)
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
                const int c = 2 * s + (lane >> 5);
                const uint32_t at = (uint32_t)(down[n] * pitch + (head[n] * d + c * V) * (int)sizeof(T));
                f[n][s] = __builtin_bit_cast(F, __builtin_amdgcn_raw_buffer_load_b128(
                                                    buffer, exists[n] && (c + 1) * V <= d ? (int)at : (int)kPastEnd, 0, 0));
            }
        if (d % V == 0) return;
        const int last = d / V;   // the chunk that the head ends in, element by element
        if ((lane >> 5) != (last & 1)) return;
#pragma unroll
        for (int n = 0; n < QB; ++n) {
            if (!exists[n]) continue;
            const T* p = (const T*)(from + down[n] * pitch) + (int64_t)head[n] * d + last * V;
            F v = {};
#pragma unroll
            for (int e = 0; e < V - 1; ++e)
                if (last * V + e < d) v[e] = p[e];
#pragma unroll
            for (int s = 0; s < STEPS; ++s)
                if (s == last / 2) f[n][s] = v;
        }
    }
};

// Eight columns from c0 on of a row's head of d columns.
template <class T>
__device__ __forceinline__ void store_eight(T* row, int c0, int d, const float (&v)[8]) {
    typedef T Eight __attribute__((ext_vector_type(8), aligned(sizeof(T))));
    if (c0 + 8 <= d) {
        Eight u;
#pragma unroll
        for (int e = 0; e < 8; ++e) u[e] = (T)v[e];
        *(Eight*)(row + c0) = u;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (c0 + e < d) row[c0 + e] = (T)v[e];
    }
}

// Registers 8 p .. 8 p + 7 of a square exchanged between the halves: the lane
// then holds rows 16 p + 8 (lane / 32) .. + 7.
__device__ __forceinline__ void square_rows(const f32x16& s, int p, float (&v)[8]) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        v[r] = s[8 * p + r];
        v[4 + r] = s[8 * p + 4 + r];
        swap32(v[r], v[4 + r]);
    }
}

// s scale log2(e), or no difference between states for a scale of 0; positive, so
// that -infinity stays -infinity.
inline float exponent_of(float scale) { return scale > 0.0f ? fmaxf(scale * kLog2E, 0x1p-149f) : 0x1p-149f; }

// The least multiple of 32 that the kernels hold heads in.
template <class F>
void by_head_width(int head, F f) {
    if (head <= 32) f(Constant<32>{});
    else if (head <= 64) f(Constant<64>{});
    else if (head <= 96) f(Constant<96>{});
    else f(Constant<128>{});
}

}  // namespace tgs
