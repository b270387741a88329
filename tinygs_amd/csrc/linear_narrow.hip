// The gradients of a narrow linear layer (rows of x and of dy up to 512 bytes:
// 256 halves, 128 floats) in one pass over the rows: dz = dy act'(z) once from
// memory, then dx = dz w and the workgroup's share of dw = dz^T x and db from
// LDS. Bound by the bytes: dy, z and x are read once and dx is written once,
// where a pass for dz and a product each for dx and dw would move 7 arrays of
// the rows instead of 4.
//
// A workgroup of eight waves, one a compute unit, walks over blocks of 32 rows.
// w stays in LDS (up to 128 KB), dw's float sums in the registers of the waves
// (128 x 64 a wave for halves); a block's dz and x take 16 KB each. The next
// block's dy, z and x are on their way into registers while a block is
// multiplied. The workgroups' sums are joined by a second kernel in a fixed
// order. 1e6 x 256 -> 256 halves with gelu: 2.05 GB in 505 us (4.1 TB/s) and the
// join of 256 sums 17 us; 50021 x 84 -> 128 floats 31 and 6 us.
#include "narrow_rows.h"

namespace tgs {

namespace {

template <class T>
struct Plane {
    using type = T;
};
template <>
struct Plane<float> {
    using type = __bf16;
};

constexpr int kRows = 32;   // of a block
// Rows after a block's, of two bytes or more each, that hold the 14 bytes which
// a partial chunk may reach past the block's last row.
constexpr int kBeyond = 8;
constexpr int kThreads = 512;

// Matrices in LDS: halves as they are, in rows of 512 bytes; floats as the
// three bfloat16 planes of split3, each of rows of 256 bytes, split once as
// they are placed.
template <class T>
struct Narrow {
    using C = Chunk<T>;
    static constexpr int V = C::V;
    static constexpr int kCols = 512 / (int)sizeof(T);
    static constexpr int kPlanes = sizeof(T) == 4 ? 3 : 1, kPitch = sizeof(T) == 4 ? 256 : 512;
    using E = typename Plane<T>::type;
    using R = NarrowRows<E, kPitch>;
    static constexpr int kSteps = kCols / 32;               // of dx's k
    static constexpr int TI = kCols / 32, TJ = kCols / 64;  // dw squares of a wave: two waves on in, four on out
    static constexpr int DI = kCols / 128;                  // dx squares of a wave on in
    static constexpr int kWeightPlane = kCols * kPitch, kBlockPlane = kRows * kPitch;
    static constexpr int kWeights = kPlanes * kWeightPlane, kBlock = kPlanes * kBlockPlane;
    static constexpr int kLds = kWeights + 2 * kBlock;
    typedef typename C::type chunk;
    typedef typename Frag<T>::type frag;

    // A chunk of row r at its place: 16 bytes, or 8 in each plane.
    static __device__ __forceinline__ void place(unsigned char* rows, int plane, int r, int c, const chunk& v) {
        if constexpr (sizeof(T) == 2) {
            *(chunk*)(rows + R::at(r, c)) = v;
        } else {
            typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
            u32x2 p[3];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float x = v[2 * e], y = v[2 * e + 1];
#pragma unroll
                for (int q = 0; q < 3; ++q) p[q][e] = take_bf16(x, y);
            }
#pragma unroll
            for (int q = 0; q < 3; ++q) *(u32x2*)(rows + q * plane + R::at(r, c / 2) + (c & 1) * 8) = p[q];
        }
    }
    static __device__ __forceinline__ frag k_fragment(const unsigned char* rows, int plane, int r0, int s, int lane) {
        if constexpr (sizeof(T) == 2) return R::k_fragment(rows, r0, s, lane);
        else return frag{R::k_fragment(rows, r0, s, lane), R::k_fragment(rows + plane, r0, s, lane),
                         R::k_fragment(rows + 2 * plane, r0, s, lane)};
    }
    static __device__ __forceinline__ frag r_fragment(const unsigned char* rows, int plane, int c0, int s, int lane) {
        if constexpr (sizeof(T) == 2) return R::r_fragment(rows, c0, s, lane);
        else return frag{R::r_fragment(rows, c0, s, lane), R::r_fragment(rows + plane, c0, s, lane),
                         R::r_fragment(rows + 2 * plane, c0, s, lane)};
    }
};

// partial + blockIdx.x * (out * in + out): the workgroup's dw and db.
// Buffer loads give zeros where nothing is, and stores there are dropped.
// RAGGED: in or out is no multiple of a chunk. A partial chunk is then loaded
// whole, with what follows in memory, and masked when it is used; the blocks
// that end the matrix, where nothing need follow, are gathered element by
// element.
template <class T, int ACT, bool RAGGED>
__global__ void __launch_bounds__(kThreads) backward_kernel(LinearBackward a, float* partial, int blocks) {
    using N = Narrow<T>;
    constexpr int V = N::V;
    __shared__ __align__(1024) unsigned char lds[N::kLds];
    unsigned char *const w = lds, *const dz = lds + N::kWeights, *const xs = dz + N::kBlock;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int in = (int)a.x.cols, out = (int)a.grad_y.cols;
    const int64_t rows = a.grad_y.rows;

    // a thread's chunk of the columns, and its rows of a block: r and r + 16
    const int chunk = tid & 31, r = tid >> 5;
    const int n_in = min(max(in - chunk * V, 0), V), n_out = min(max(out - chunk * V, 0), V);

    // A matrix's 32 rows (from `first` on) as this thread's two chunks.
    const auto load = [&](const Mat& m, int64_t first, int n, typename N::chunk(&to)[2]) {
        const T* base = (const T*)m.p + first * m.stride;
        const int64_t pitch = m.stride * (int64_t)sizeof(T);
        // rows beyond the block's lie between it and the buffer's end when a chunk may reach past a row
        const int64_t held = min(m.rows - first, (int64_t)(RAGGED ? kRows + kBeyond : kRows));
        const auto buffer = resource_of(base, RAGGED && held < kRows + kBeyond
                                                  ? 0 : (held - 1) * pitch + m.cols * (int64_t)sizeof(T));
        const uint32_t from = (n > 0 ? 0u : kNowhere) + (uint32_t)chunk * 16u;
#pragma unroll
        for (int h = 0; h < 2; ++h)
            to[h] = __builtin_bit_cast(typename N::chunk, __builtin_amdgcn_raw_buffer_load_b128(
                                                              buffer, (int)(from + (uint32_t)(r + 16 * h) * (uint32_t)pitch), 0, 0));
    };
    // Ahead of their use, RAGGED: chunks that load left out or loaded more than is there.
    const auto mend = [&](const Mat& m, int64_t first, int n, typename N::chunk(&v)[2]) {
        if constexpr (!RAGGED) return;
        if (m.rows - first < kRows + kBeyond) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int row = r + 16 * h;
                const bool exists = first + row < m.rows && n > 0;
                v[h] = N::C::gather(exists ? (const T*)m.p + (first + row) * m.stride + chunk * V : (const T*)m.p,
                                    exists ? n : 0);
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int e = 0; e < V; ++e) v[h][e] = e < n ? v[h][e] : (T)0.0f;
    };

    typename N::chunk dy[2], z[2], x[2];
    const auto fetch_block = [&](int block) {
        const int64_t first = (int64_t)block * kRows;
        load(a.grad_y, first, n_out, dy);
        if constexpr (ACT != kActNone) load(a.preact, first, n_out, z);
        if (a.grad_w.p) load(a.x, first, n_in, x);
    };

    fetch_block(blockIdx.x);
    const bool deep = out > N::kCols / 2;
    if (a.grad_x.p) {   // zeros past out, up to the half that dx reads
        constexpr int kQuarters = N::kCols / kRows / 2;
        const auto place = [&](int n0) {
            typename N::chunk v[kQuarters][2];
#pragma unroll
            for (int q = 0; q < kQuarters; ++q) load(a.w, n0 + kRows * q, n_in, v[q]);
#pragma unroll
            for (int q = 0; q < kQuarters; ++q) {
                mend(a.w, n0 + kRows * q, n_in, v[q]);
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    N::place(w, N::kWeightPlane, n0 + kRows * q + r + 16 * h, chunk, v[q][h]);
            }
        };
        place(0);
        if (deep) place(N::kCols / 2);
    }

    f32x4 acc[N::TI][N::TJ];
#pragma unroll
    for (int u = 0; u < N::TI; ++u)
#pragma unroll
        for (int v = 0; v < N::TJ; ++v) acc[u][v] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float sum[V] = {};
    const int wi = wave >> 2, wj = wave & 3;
    const bool dw_here = a.grad_w.p && wi * N::TI * 16 < in && wj * N::TJ * 16 < out;
    const bool dx_here = a.grad_x.p && wave * N::DI * 16 < in;
    const auto slope_of = [&](int64_t row, int column) {   // dz as form_again reads it
        if (row >= rows || column >= out) return 0.0f;
        const float d = (float)((const T*)a.grad_y.p)[row * a.grad_y.stride + column];
        if constexpr (ACT == kActNone) return d;
        else return d * activate_slope<ACT>((float)((const T*)a.preact.p)[row * a.preact.stride + column]);
    };

    for (int block = blockIdx.x; block < blocks; block += gridDim.x) {
        lds_barrier();   // the last block's reads are done
        if constexpr (RAGGED) {
            const int64_t first = (int64_t)block * kRows;
            mend(a.grad_y, first, n_out, dy);
            if constexpr (ACT != kActNone) mend(a.preact, first, n_out, z);   // no NaN against a zero of dy
            if (a.grad_w.p) mend(a.x, first, n_in, x);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if constexpr (ACT != kActNone) {
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float d = (float)dy[h][e] * activate_slope<ACT>((float)z[h][e]);
                    sum[e] += d;
                    dy[h][e] = (T)d;   // halves: one operand of the products, and all that LDS has room for beside w
                }
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e) sum[e] += (float)dy[h][e];
            }
            N::place(dz, N::kBlockPlane, r + 16 * h, chunk, dy[h]);
            if (a.grad_w.p) N::place(xs, N::kBlockPlane, r + 16 * h, chunk, x[h]);
        }
        lds_barrier();
        if (block + (int)gridDim.x < blocks) fetch_block(block + gridDim.x);

        // The addresses below are formed anew for each block: kept over the
        // blocks they would take the registers of the sums.
        int near = lane;
        asm volatile("" : "+v"(near));
        if (dx_here) {
            f32x4 d[N::DI][2];
#pragma unroll
            for (int u = 0; u < N::DI; ++u) d[u][0] = d[u][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            typename N::frag fw[2][N::DI], fz[2][2];
            const auto read = [&](int s, int to) {
#pragma unroll
                for (int u = 0; u < N::DI; ++u) fw[to][u] = N::r_fragment(w, N::kWeightPlane, (wave * N::DI + u) * 16, s, near);
#pragma unroll
                for (int v = 0; v < 2; ++v) fz[to][v] = N::k_fragment(dz, N::kBlockPlane, 16 * v, s, near);
            };
            const auto half = [&](int s0) {
                read(s0, 0);
#pragma unroll
                for (int s = 0; s < N::kSteps / 2; ++s) {
                    if (s < N::kSteps / 2 - 1) read(s0 + s + 1, (s + 1) & 1);
#pragma unroll
                    for (int u = 0; u < N::DI; ++u)
#pragma unroll
                        for (int v = 0; v < 2; ++v) d[u][v] = multiply(fw[s & 1][u], fz[s & 1][v], d[u][v]);
                }
            };
            half(0);
            if (deep) half(N::kSteps / 2);
            if constexpr (sizeof(T) == 4)
                form_again(
                    d, 0, out,
                    [&](int u, int row, int64_t k) {
                        const int i = (wave * N::DI + u) * 16 + row;
                        return i < in ? ((const T*)a.w.p)[k * a.w.stride + i] : 0.0f;
                    },
                    [&](int v, int row, int64_t k) { return slope_of((int64_t)block * kRows + 16 * v + row, (int)k); },
                    [](int, int, int) { return true; });
            const int64_t first = (int64_t)block * kRows, pitch = a.grad_x.stride * (int64_t)sizeof(T);
            T* const base = (T*)a.grad_x.p + first * a.grad_x.stride;
            const auto buffer = resource_of(base, (min(rows - first, (int64_t)kRows) - 1) * pitch + in * (int64_t)sizeof(T));
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                const int row = 16 * v + (lane & 15);
                int i;
                typename N::chunk y;
                if constexpr (N::DI == 2) {
                    float f[8];
                    neighbours(d[0][v], d[1][v], f);
                    i = wave * 32 + neighbours_at(lane);
#pragma unroll
                    for (int e = 0; e < V; ++e) y[e] = (T)f[e];
                } else {
                    i = wave * 16 + 4 * (lane >> 4);
#pragma unroll
                    for (int e = 0; e < V; ++e) y[e] = (T)d[0][v][e];
                }
                if constexpr (!RAGGED) {
                    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, y), buffer,
                                                           (int)((i < in ? 0u : kNowhere) + (uint32_t)row * (uint32_t)pitch + (uint32_t)i * (uint32_t)sizeof(T)),
                                                           0, 0);
                } else if (first + row < rows && i + V <= in) {
                    typedef T loose __attribute__((ext_vector_type(V), aligned(sizeof(T))));
                    *(loose*)(base + row * a.grad_x.stride + i) = __builtin_bit_cast(loose, y);
                } else if (first + row < rows) {
#pragma unroll
                    for (int e = 0; e < V; ++e)
                        if (i + e < in) base[row * a.grad_x.stride + i + e] = y[e];
                }
            }
        }
        if (dw_here) {
            typename N::frag fz[N::TJ];
#pragma unroll
            for (int v = 0; v < N::TJ; ++v) fz[v] = N::r_fragment(dz, N::kBlockPlane, (wj * N::TJ + v) * 16, 0, near);
#pragma unroll
            for (int u = 0; u < N::TI; ++u) {
                if (u >= N::TI / 2 && (wi * N::TI + u) * 16 >= in) break;
                const auto fx = N::r_fragment(xs, N::kBlockPlane, (wi * N::TI + u) * 16, 0, near);
#pragma unroll
                for (int v = 0; v < N::TJ; ++v) acc[u][v] = multiply(fx, fz[v], acc[u][v]);
            }
        }
    }

    float* to = partial + (int64_t)blockIdx.x * ((int64_t)out * in + out);
    if constexpr (sizeof(T) == 4)
        if (dw_here) {   // k runs over the rows of the workgroup's blocks
            const int own = (blocks - 1 - (int)blockIdx.x) / (int)gridDim.x + 1;
            const auto row_of = [&](int64_t k) {
                return ((int64_t)blockIdx.x + (k / kRows) * gridDim.x) * kRows + k % kRows;
            };
            form_again(
                acc, 0, (int64_t)own * kRows,
                [&](int u, int row, int64_t k) {
                    const int64_t r = row_of(k);
                    const int i = (wi * N::TI + u) * 16 + row;
                    return r < rows && i < in ? ((const T*)a.x.p)[r * a.x.stride + i] : 0.0f;
                },
                [&](int v, int row, int64_t k) { return slope_of(row_of(k), (wj * N::TJ + v) * 16 + row); },
                [](int, int, int) { return true; });
        }
    if (dw_here) {
        const auto buffer = resource_of(to, (int64_t)out * in * 4);   // at most 256 KB
        const bool fours = in % 4 == 0;
#pragma unroll
        for (int u = 0; u < N::TI; ++u) {
            const int i = (wi * N::TI + u) * 16 + 4 * (lane >> 4);
#pragma unroll
            for (int v = 0; v < N::TJ; ++v) {
                const int j = (wj * N::TJ + v) * 16 + (lane & 15);
                const uint32_t at = (uint32_t)(j * in + i) * 4u;
                if (fours) {
                    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, acc[u][v]), buffer,
                                                           (int)(at + (i < in ? 0u : kNowhere)), 0, 0);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float f = acc[u][v][e];
                        __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, f), buffer,
                                                              (int)(at + 4u * e + (i + e < in ? 0u : kNowhere)), 0, 0);
                    }
                }
            }
        }
    }
    if (a.grad_bias) {   // the sixteen threads of a chunk, in order
        float* s = (float*)lds;
        lds_barrier();
#pragma unroll
        for (int e = 0; e < V; ++e) s[r * N::kCols + chunk * V + e] = sum[e];
        lds_barrier();
        for (int k = tid; k < out; k += kThreads) {
            float v = s[k];
            for (int q = 1; q < 16; ++q) v += s[q * N::kCols + k];
            to[(int64_t)out * in + k] = v;
        }
    }
}

}  // namespace

// Against a slope pass and two tile products, us, with SiLU: 1e6 x 256 -> 256
// halves 510 and 779, 1e6 x 128 -> 128 289 and 366, 100000 rows 44 and 55, 2000 x
// 72 -> 72 16 and 22, 1e6 x 128 -> 64 283 and 260; floats 1e6 x 128 -> 64 400 and
// 550, 2000 rows 18 and 43.
// A block of 32 rows takes its 2 us however few columns it has, so that many
// rows of few (in and out together up to 256 bytes) are tiles' sooner: halves
// 1e6 x 32 -> 32 249 and 113, 64 -> 64 254 and 189, 3 -> 64 373 and 163, 59 -> 3
// 343 and 148; 200000 rows 59 and 42, 62 and 51, 89 and 51, 84 and 51, without an
// activation at worst 61 and 67 (63 -> 59); 100000 rows 36 and 32, 37 and 37, 54
// and 35, 53 and 40, at worst 36 and 43 (16 -> 112). Floats, whose tiles are six
// products: 1e6 x 32 -> 32 265 and 206, 2 -> 32 333 and 207, 8 -> 56 265 and 282;
// 400000 rows 113 and 99, 141 and 102, 113 and 129; 200000 rows 63 and 69, 78 and
// 69, 63 and 84.
// Ragged halves of more than 128 columns take their last rows of w element by
// element, which fewer rows do not pay back: 250 -> 256, 2000 rows 50 and 28 us,
// 20000 62 and 41, 200000 178 and 216.
bool linear_backward_is_narrow(const LinearBackward& a) {
    const bool floats = a.dtype == TGS_DTYPE_FLOAT32;
    const int64_t size = floats ? 4 : 2, most = 512 / size, in = a.x.cols, out = a.grad_y.cols, rows = a.grad_y.rows;
    if (!floats && (in % 8 || out % 8) && in > 128 && out > 128 && rows < 65536) return false;
    if ((in + out) * size <= 256 && rows >= (floats ? 300000 : 200000)) return false;
    return in <= most && out <= most && rows > 0;
}

int narrow_backward_splits(const LinearBackward& a) {
    // a workgroup's sums are worth four blocks; no more workgroups than compute units
    const int64_t want = (a.grad_y.rows + 4 * kRows - 1) / (4 * kRows);
    return (int)(want < 256 ? want : 256);
}

void launch_narrow_backward(const LinearBackward& a, float* partial, hipStream_t s) {
    const int blocks = (int)((a.grad_y.rows + kRows - 1) / kRows);
    by_dtype(a.dtype, [&](auto t) {
        by_activation(a.activation, [&](auto act) {
            using T = decltype(t);
            constexpr int kAct = decltype(act)::value;
            if (a.x.cols % Chunk<T>::V || a.grad_y.cols % Chunk<T>::V)
                backward_kernel<T, kAct, true><<<narrow_backward_splits(a), kThreads, 0, s>>>(a, partial, blocks);
            else
                backward_kernel<T, kAct, false><<<narrow_backward_splits(a), kThreads, 0, s>>>(a, partial, blocks);
        });
    });
}

}  // namespace tgs
