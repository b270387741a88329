// LDS rows of 256 or 512 bytes for the narrow linear layers' kernels. A row's
// 16-byte chunks are permuted by the row, so that both reads are free of bank
// conflicts: 16 rows at one chunk (K-contiguous), and runs of 16 halves of 4
// rows at a time (R-contiguous).
#pragma once

#include "mfma_tile.h"

namespace tgs {

// Past the end of every block of up to 64 rows (of less than 2^23 bytes each),
// also with an offset within the block added, and that below 2^32.
constexpr uint32_t kNowhere = 0xc0000000u;

template <class T>
struct Chunk {
    static constexpr int V = 16 / (int)sizeof(T);   // elements of 16 bytes
    typedef T type __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));

    // n (0 to V) elements at p, zeros after them; p is readable where n is 0.
    static __device__ __forceinline__ type gather(const T* p, int n) {
        type v;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const T u = p[min(e, max(n - 1, 0))];
            v[e] = e < n ? u : (T)0.0f;
        }
        return v;
    }
};

template <class T, int PITCH>
struct NarrowRows {
    static_assert(PITCH == 256 || PITCH == 512, "sixteen or thirty-two chunks");
    static constexpr int kCols = PITCH / (int)sizeof(T);

    // Sixteen rows take all sixteen chunk slots; the rows 8 g + q of one
    // R-contiguous read take different runs.
    static __device__ __forceinline__ int turn(int r) { return ((r & 3) << 1) | ((r >> 2) & 1) | (r & 8); }
    static __device__ __forceinline__ int at(int r, int chunk) { return r * PITCH + ((chunk ^ turn(r)) << 4); }

    // Elements 32 s .. + 31 of rows r0 .. r0 + 15 (r0 a multiple of 16).
    static __device__ __forceinline__ typename Frag<T>::type k_fragment(const unsigned char* rows, int r0, int s, int lane) {
        const int a = lane & 15, g = lane >> 4;
        if constexpr (sizeof(T) == 4) {
            float x[8];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const f32x4 v = *(const f32x4*)(rows + at(r0 + a, 8 * s + 2 * g + h));
#pragma unroll
                for (int e = 0; e < 4; ++e) x[4 * h + e] = v[e];
            }
            return split3(x);
        } else {
            return *(const typename Frag<T>::type*)(rows + at(r0 + a, 4 * s + g));
        }
    }

    // Columns c0 .. c0 + 15 of rows 32 s .. + 31.
    static __device__ __forceinline__ typename Frag<T>::type r_fragment(const unsigned char* rows, int c0, int s, int lane) {
        static_assert(sizeof(T) == 2, "halves only");
        const int a = lane & 15, g = lane >> 4;
        const int q = a >> 2, k = 32 * s + 8 * g + q, chunk = c0 / 8 + ((a & 3) >> 1), in = (a & 1) * 8;
        typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
        union {
            i16x4 half[2];
            typename Frag<T>::type whole;
        } u;
        u.half[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(lds_byte*)(rows + at(k, chunk) + in));
        u.half[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(lds_byte*)(rows + at(k + 4, chunk) + in));
        return u.whole;
    }
};

}  // namespace tgs
