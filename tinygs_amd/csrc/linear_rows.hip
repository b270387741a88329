// y = act(x w^T + bias) + residual for many rows of a narrow layer (rows of x
// up to 512 bytes: 256 halves, 128 floats), bound by the bytes of x, residual,
// preact and y.
//
// w stays in registers: each of a workgroup's eight waves holds the fragments
// of its columns (32 halves or 16 floats wide) for all of k, and the workgroup
// walks over blocks of 64 rows, so that w is read once a workgroup and not once
// a tile. x and the residual come to LDS without passing registers, the next
// block's while the current one is multiplied; the wait for them leaves the
// stores of the block before in flight. 1e6 x 256 -> 256 halves with gelu,
// residual and preact: 2.05 GB.
#include "narrow_rows.h"

namespace tgs {

namespace {

constexpr int kRows = 64;
constexpr int kThreads = 512;

// PITCH: bytes of a row of x in LDS. CW waves share the columns (COLS of them
// a workgroup), 8 / CW the rows.
template <class T, int PITCH, int CW, bool RESIDUAL>
struct RowsKernel {
    using X = NarrowRows<T, PITCH>;
    static constexpr int V = X::V;
    static constexpr int kSquares = 32 / (int)sizeof(T) / 8;      // of columns a wave: 2 (halves), 1 (floats)
    static constexpr int kCols = CW * kSquares * 16;
    static constexpr int kResidualPitch = CW * 64;                // bytes of kCols elements
    using R = NarrowRows<T, kResidualPitch>;
    static constexpr int kRowSquares = 4 * CW / 8;                // of rows a wave
    static constexpr int kSteps = PITCH / 64;
    static constexpr int kXBytes = kRows * PITCH, kStage = kXBytes + (RESIDUAL ? kRows * kResidualPitch : 0);
    static constexpr int kLds = 2 * kStage;

    // Rows `first` .. + 63 of m from column c0 on, as rows of PITCH2 bytes in
    // LDS. Chunks past m's columns are filled from what follows in memory,
    // which its user masks or ignores; the chunk that crosses the matrix's end
    // is gathered (`last`: the block holds the last row).
    template <class F>
    static __device__ __forceinline__ void load(const Mat& m, int64_t first, int64_t c0, unsigned char* lds, bool last,
                                                int wave, int lane) {
        constexpr int kChunks = F::kCols / V, kLoads = kRows * kChunks / 64 / 8;
        const int64_t pitch = m.stride * (int64_t)sizeof(T);
        const T* base = (const T*)m.p + first * m.stride + c0;
        const int64_t rows = min(m.rows - first, (int64_t)kRows);
        const int cols = (int)min(m.cols - c0, (int64_t)F::kCols);
        const int tail = cols % V;   // elements of a partial chunk
        // whole chunks beyond the columns are left out; a partial one of an inner row may be read whole
        const i32x4 buffer = buffer_of(base, (rows - 1) * pitch + (int64_t)(tail && !last ? cols - tail + V : cols) * (int64_t)sizeof(T));
        const uint32_t to = lds_address(lds);
#pragma unroll
        for (int n = 0; n < kLoads; ++n) {
            const int slot = (n * 8 + wave) * 64 + lane, r = slot / kChunks, c = (slot % kChunks) ^ F::turn(r);
            const uint32_t offset = (c * V < cols ? 0u : kNowhere) + (uint32_t)r * (uint32_t)pitch + (uint32_t)c * 16u;
            if (tail && last && c == cols / V) {
                const T* p = base + (r < rows ? r : 0) * m.stride + c * V;
                const auto v = F::gather(p, r < rows ? tail : 0);
                *(typename F::loose*)(lds + slot * 16) = v;
            } else {
                load_to_lds(to + (n * 8 + wave) * 1024, offset, buffer);
            }
        }
    }
};

template <int ACT>
__device__ __forceinline__ void activate_all(float (&v)[8], int n) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (e < n) v[e] = activate<ACT>(v[e]);
}

template <class T, int PITCH, int CW, bool RESIDUAL>
__global__ void __launch_bounds__(kThreads) rows_kernel(LinearForward a, int blocks) {
    using K = RowsKernel<T, PITCH, CW, RESIDUAL>;
    using X = typename K::X;
    constexpr int V = K::V;
    __shared__ __align__(1024) unsigned char lds[K::kLds];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wc = wave % CW, wr = wave / CW;
    const int in = (int)a.x.cols;
    const int64_t out = a.y.cols, rows = a.y.rows, c0 = (int64_t)blockIdx.y * K::kCols;
    const Mat residual = a.residual;

    const auto load = [&](int block) {
        const int64_t first = (int64_t)block * kRows;
        unsigned char* stage = lds + ((block / gridDim.x) & 1) * K::kStage;
        const bool last = first + kRows >= rows;
        K::template load<X>(a.x, first, 0, stage, last, wave, lane);
        if constexpr (RESIDUAL) K::template load<typename K::R>(residual, first, c0, stage + K::kXBytes, last, wave, lane);
    };
    load(blockIdx.x);

    // w's fragments: columns c of y are rows of w
    const int64_t column0 = c0 + wc * K::kSquares * 16;
    typename Frag<T>::type fw[K::kSquares][K::kSteps];
#pragma unroll
    for (int u = 0; u < K::kSquares; ++u)
#pragma unroll
        for (int s = 0; s < K::kSteps; ++s) {
            const int64_t n = column0 + 16 * u + (lane & 15);
            const int k = s * X::kHalf + (lane >> 4) * V;
            const int left = n < out ? min(max(in - k, 0), V) : 0;
            const T* p = (const T*)a.w.p + (n < out ? n : 0) * a.w.stride + (left > 0 ? k : 0);
            if (in % V == 0) {
                const auto v = *(const typename X::loose*)p;   // left is 0 or V; a whole chunk of row n or 0 is there
#pragma unroll
                for (int e = 0; e < V; ++e) fw[u][s][e] = left > 0 ? v[e] : (T)0.0f;
            } else {
                const auto v = X::gather(p, left);
#pragma unroll
                for (int e = 0; e < V; ++e) fw[u][s][e] = v[e];
            }
        }
    // a lane's run of V outputs: columns at .. at + V - 1 of y
    const int64_t at = column0 + (K::kSquares == 2 ? neighbours_at(lane) : 4 * (lane >> 4));
    const int exist = (int)min(max(out - at, (int64_t)0), (int64_t)V);
    float bias[V];
#pragma unroll
    for (int e = 0; e < V; ++e) bias[e] = a.bias && e < exist ? a.bias[at + e] : 0.0f;
    // The chunk of x that ends k: lanes that hold it clear what follows.
    const int tail = in % V, tail_step = in / X::kHalf;
    const bool clears = tail && (lane >> 4) == in % X::kHalf / V;

    const bool ragged = out % V != 0;
    // a block's stores: these many at least are issued after the next block's loads
    const int stores = ragged ? 0 : K::kRowSquares * (a.preact.p ? 2 : 1);
    bool stored = false;
    for (int block = blockIdx.x; block < blocks; block += gridDim.x) {
        // this block's loads are done when no more are in flight than the stores after them
        if (!stored || stores == 0) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        else if (stores == K::kRowSquares) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(K::kRowSquares) : "memory");
        else asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(2 * K::kRowSquares) : "memory");
        stored = true;
        if (block + (int)gridDim.x < blocks) load(block + gridDim.x);

        const unsigned char* stage = lds + ((block / gridDim.x) & 1) * K::kStage;
        f32x4 acc[K::kSquares][K::kRowSquares];
#pragma unroll
        for (int u = 0; u < K::kSquares; ++u)
#pragma unroll
            for (int v = 0; v < K::kRowSquares; ++v) acc[u][v] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int s = 0; s < K::kSteps; ++s) {
            if (s == K::kSteps / 2 && in <= s * X::kHalf) break;   // w is zero there
            typename Frag<T>::type fx[K::kRowSquares];
#pragma unroll
            for (int v = 0; v < K::kRowSquares; ++v) {
                fx[v] = X::k_fragment(stage, (wr * K::kRowSquares + v) * 16, s, lane);
                if (s == tail_step && tail)
#pragma unroll
                    for (int e = 0; e < V; ++e) fx[v][e] = clears && e >= tail ? (T)0.0f : fx[v][e];
            }
#pragma unroll
            for (int u = 0; u < K::kSquares; ++u)
#pragma unroll
                for (int v = 0; v < K::kRowSquares; ++v) acc[u][v] = multiply(fw[u][s], fx[v], acc[u][v]);
        }

        const int64_t first = (int64_t)block * kRows;
        const int64_t held = min(rows - first, (int64_t)kRows) - 1;
        const int64_t y_pitch = a.y.stride * (int64_t)sizeof(T), z_pitch = a.preact.stride * (int64_t)sizeof(T);
        T* const y0 = (T*)a.y.p + first * a.y.stride + at;
        T* const z0 = (T*)a.preact.p + first * a.preact.stride + at;
        const auto y_buffer = resource_of((T*)a.y.p + first * a.y.stride, held * y_pitch + out * (int64_t)sizeof(T));
        const auto z_buffer = resource_of((T*)a.preact.p + first * a.preact.stride, held * z_pitch + out * (int64_t)sizeof(T));
#pragma unroll
        for (int v = 0; v < K::kRowSquares; ++v) {
            const int r = (wr * K::kRowSquares + v) * 16 + (lane & 15);
            float f[8];
            if constexpr (K::kSquares == 2) {
                neighbours(acc[0][v], acc[1][v], f);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) f[e] = acc[0][v][e];
            }
#pragma unroll
            for (int e = 0; e < V; ++e) f[e] += bias[e];
            const auto store = [&](const __amdgpu_buffer_rsrc_t& buffer, T* p, int64_t stride, int64_t pitch) {
                typename X::loose o;
#pragma unroll
                for (int e = 0; e < V; ++e) o[e] = (T)f[e];
                if (!ragged) {
                    __builtin_amdgcn_raw_buffer_store_b128(
                        __builtin_bit_cast(u32x4, o), buffer,
                        (int)((exist > 0 ? 0u : kNowhere) + (uint32_t)r * (uint32_t)pitch + (uint32_t)at * (uint32_t)sizeof(T)), 0, 0);
                } else if (r <= held) {
#pragma unroll
                    for (int e = 0; e < V; ++e)
                        if (e < exist) p[r * stride + e] = o[e];
                }
            };
            if (a.preact.p) store(z_buffer, z0, a.preact.stride, z_pitch);
            if (a.activation == kActGelu) activate_all<kActGelu>(f, V);
            else if (a.activation == kActSilu) activate_all<kActSilu>(f, V);
            else if (a.activation == kActRelu) activate_all<kActRelu>(f, V);
            if constexpr (RESIDUAL) {
                const auto q = *(const typename X::loose*)(stage + K::kXBytes + K::R::at(r, (int)(at - c0) / V));
#pragma unroll
                for (int e = 0; e < V; ++e) f[e] += (float)q[e];
            }
            store(y_buffer, y0, a.y.stride, y_pitch);
        }
    }
}

}  // namespace

bool linear_forward_by_rows(const LinearForward& a) {
    const int64_t most = 512 / (a.dtype == TGS_DTYPE_FLOAT32 ? 4 : 2);
    return a.x.cols <= most && a.y.cols <= 4 * most && a.y.rows >= 4096;
}

void launch_linear_rows(const LinearForward& a, hipStream_t s) {
    const int blocks = (int)((a.y.rows + kRows - 1) / kRows);
    by_dtype(a.dtype, [&](auto t) {
        using T = decltype(t);
        constexpr int kMost = 512 / (int)sizeof(T);
        const auto launch = [&](auto pitch, auto cw, auto residual) {
            constexpr int P = decltype(pitch)::value, CW = decltype(cw)::value;
            constexpr bool kResidual = decltype(residual)::value != 0;
            using K = RowsKernel<T, P, CW, kResidual>;
            // as many workgroups as the card holds at once
            constexpr int kResident = 160 * 1024 / K::kLds < 2 ? 1 : 2;
            const int across = (int)((a.y.cols + K::kCols - 1) / K::kCols);
            const int want = 256 * kResident / across, down = blocks < want ? blocks : want;
            rows_kernel<T, P, CW, kResidual><<<dim3((unsigned)down, (unsigned)across), kThreads, 0, s>>>(a, blocks);
        };
        const auto by_residual = [&](auto pitch, auto cw) {
            if (a.residual.p) launch(pitch, cw, Constant<1>{});
            else launch(pitch, cw, Constant<0>{});
        };
        const auto by_columns = [&](auto pitch) {
            if (a.y.cols <= kMost / 2) by_residual(pitch, Constant<4>{});
            else by_residual(pitch, Constant<8>{});
        };
        if (a.x.cols <= kMost / 2) by_columns(Constant<256>{});
        else by_columns(Constant<512>{});
    });
}

}  // namespace tgs
