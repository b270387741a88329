// y = act(x w^T + bias) + residual for many rows of a narrow layer (rows of x
// up to 512 bytes: 256 halves, 128 floats), bound by the bytes of x, residual,
// preact and y.
//
// w stays in registers: each of a workgroup's eight waves holds the fragments
// of its 32 columns for all of k, and the workgroup
// walks over blocks of 64 rows, so that w is read once a workgroup and not once
// a tile. x and the residual come to LDS without passing registers, one to three
// blocks ahead; the wait for a block leaves the loads and stores that were
// started after it in flight. 1e6 x 256 -> 256 halves with gelu, residual and
// preact: 2.05 GB in 384 us, 5.3 TB/s.
#include "narrow_rows.h"

namespace tgs {

namespace {

constexpr int kRows = 64;
constexpr int kThreads = 512;

// Workgroups a compute unit holds: two where w's registers allow it.
constexpr int resident(int size, int pitch, int cw) { return size == 2 && pitch == 256 && cw <= 4 ? 2 : 1; }

// What a block's loads may read of a matrix from the block's first element on:
// `bytes`, which never pass the matrix's end. A row's partial last chunk is
// read whole, with up to 14 bytes of what follows, where the `left` rows from
// the block's first on hold as much after the block (`whole`: rows of a few
// elements need several of them), and else gathered.
struct Reach {
    bool whole;
    int bytes;   // below 2^30
};
__host__ __device__ inline Reach reach_of(int64_t left, int cols, int stride, int size) {
    const int near = left < 2 * kRows ? (int)left : 2 * kRows, held = near < kRows ? near : kRows;
    const int chunk = 16 / size, tail = cols % chunk;
    const bool whole = tail == 0 || chunk - tail <= (near - held) * stride;
    return {whole, ((held - 1) * stride + (tail && whole ? cols - tail + chunk : cols)) * size};
}

// PITCH: bytes of a row of x in LDS. CW waves share the columns (COLS of them
// a workgroup), 8 / CW the rows.
template <class T, int PITCH, int CW, bool RESIDUAL>
struct RowsKernel {
    using X = NarrowRows<T, PITCH>;
    using C = Chunk<T>;
    static constexpr int V = C::V;
    static constexpr int kCols = CW * 32;                         // two squares a wave
    static constexpr int kResidualPitch = kCols * (int)sizeof(T) < 256 ? 256 : kCols * (int)sizeof(T);
    using R = NarrowRows<T, kResidualPitch>;
    static constexpr int kRowSquares = 4 * CW / 8;                // of rows a wave
    static constexpr int kStores = kRowSquares * 8 / V;           // of y a wave and block
    static constexpr int kSteps = X::kCols / 32;
    static constexpr int kXBytes = kRows * PITCH, kStage = kXBytes + (RESIDUAL ? kRows * kResidualPitch : 0);
    static constexpr int kResident = resident((int)sizeof(T), PITCH, CW);
    static constexpr int kStages = 160 * 1024 / kResident / kStage < 4 ? 160 * 1024 / kResident / kStage : 4;
    static_assert(kStages >= 2, "two stages at least");
    static constexpr int kLds = kStages * kStage;
    static constexpr int kLoads = kStage / 1024 / 8;              // a wave and block

    // Rows `first` .. + 63 of m from column c0 on, as rows of F's pitch in
    // LDS. Chunks past m's columns are filled from what follows in memory,
    // which its user masks or ignores.
    template <class F>
    static __device__ __forceinline__ void load(const Mat& m, int64_t first, int64_t c0, unsigned char* lds, int wave,
                                                int lane) {
        constexpr int kChunks = F::kCols / V, kLoads = kRows * kChunks / 64 / 8;
        const int64_t pitch = m.stride * (int64_t)sizeof(T);
        const T* base = (const T*)m.p + first * m.stride + c0;
        const int64_t rows = min(m.rows - first, (int64_t)kRows);
        const int cols = (int)min(m.cols - c0, (int64_t)F::kCols);
        const int tail = cols % V;   // elements of a partial chunk
        const Reach reach = reach_of(m.rows - first, cols, (int)m.stride, (int)sizeof(T));
        const i32x4 buffer = buffer_of(base, reach.bytes);
        const uint32_t to = lds_address(lds);
#pragma unroll
        for (int n = 0; n < kLoads; ++n) {
            const int slot = (n * 8 + wave) * 64 + lane, r = slot / kChunks, c = (slot % kChunks) ^ F::turn(r);
            const uint32_t offset = (c * V < cols ? 0u : kNowhere) + (uint32_t)r * (uint32_t)pitch + (uint32_t)c * 16u;
            if (!reach.whole && c == cols / V) {
                const T* p = base + (r < rows ? r : 0) * m.stride + c * V;
                *(typename C::type*)(lds + slot * 16) = C::gather(p, r < rows ? tail : 0);
            } else {
                load_to_lds(to + (n * 8 + wave) * 1024, offset, buffer);
            }
        }
    }
};

template <int ACT>
__device__ __forceinline__ void activate_all(float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = activate<ACT>(v[e]);
}

// Waits until at most n of the wave's memory operations are in flight (rounded
// down to what there is an instruction for), then for the workgroup.
__device__ __forceinline__ void wait_but_for(int n) {
#define TGS_WAIT(N) \
    case N / 4: asm volatile("s_waitcnt vmcnt(" #N ") lgkmcnt(0)" ::: "memory"); break;
    switch (n / 4) {
        TGS_WAIT(0) TGS_WAIT(4) TGS_WAIT(8) TGS_WAIT(12) TGS_WAIT(16) TGS_WAIT(20) TGS_WAIT(24) TGS_WAIT(28)
        TGS_WAIT(32) TGS_WAIT(36) TGS_WAIT(40) TGS_WAIT(44) TGS_WAIT(48) TGS_WAIT(52) TGS_WAIT(56)
        default: asm volatile("s_waitcnt vmcnt(60) lgkmcnt(0)" ::: "memory");
    }
#undef TGS_WAIT
    asm volatile("s_barrier" ::: "memory");
}

template <class T, int PITCH, int CW, bool RESIDUAL>
__global__ void __launch_bounds__(kThreads, 2 * resident((int)sizeof(T), PITCH, CW)) rows_kernel(LinearForward a, int blocks) {
    using K = RowsKernel<T, PITCH, CW, RESIDUAL>;
    using X = typename K::X;
    constexpr int V = K::V;
    __shared__ __align__(1024) unsigned char lds[K::kLds];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wc = wave % CW, wr = wave / CW;
    const int in = (int)a.x.cols;
    const int64_t out = a.y.cols, rows = a.y.rows, c0 = (int64_t)blockIdx.y * K::kCols;
    const Mat residual = a.residual;

    int filled = 0;   // the stage that the next load fills
    const auto load = [&](int block) {
        const int64_t first = (int64_t)block * kRows;
        unsigned char* stage = lds + filled * K::kStage;
        filled = filled + 1 < K::kStages ? filled + 1 : 0;
        K::template load<X>(a.x, first, 0, stage, wave, lane);
        if constexpr (RESIDUAL) K::template load<typename K::R>(residual, first, c0, stage + K::kXBytes, wave, lane);
    };
#pragma unroll
    for (int n = 0; n < K::kStages - 1; ++n)
        if ((int)(blockIdx.x + n * gridDim.x) < blocks) load(blockIdx.x + n * gridDim.x);

    // w's fragments: columns c of y are rows of w
    const int64_t column0 = c0 + wc * 32;
    typename Frag<T>::type fw[2][K::kSteps];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int s = 0; s < K::kSteps; ++s) {
            const int64_t n = column0 + 16 * u + (lane & 15);
            T x[8];
#pragma unroll
            for (int h = 0; h < 8 / V; ++h) {
                const int k = 32 * s + 8 * (lane >> 4) + V * h;
                const int left = n < out ? min(max(in - k, 0), V) : 0;
                const T* p = (const T*)a.w.p + (n < out ? n : 0) * a.w.stride + (left > 0 ? k : 0);
                typename K::C::type v;
                if (in % V == 0) {   // left is 0 or V, and row n or 0 has a whole chunk
                    v = *(const typename K::C::type*)p;
#pragma unroll
                    for (int e = 0; e < V; ++e) v[e] = left > 0 ? v[e] : (T)0.0f;
                } else {
                    v = K::C::gather(p, left);
                }
#pragma unroll
                for (int e = 0; e < V; ++e) x[V * h + e] = v[e];
            }
            if constexpr (sizeof(T) == 4) {
                fw[u][s] = split3(x);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) fw[u][s][e] = x[e];
            }
        }
    // a lane's run of 8 outputs: columns at .. at + 7 of y
    const int64_t at = column0 + neighbours_at(lane);
    const int exist = (int)min(max(out - at, (int64_t)0), (int64_t)8);
    float bias[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) bias[e] = a.bias && e < exist ? a.bias[at + e] : 0.0f;
    // Elements of x past k in the chunk that ends it are whatever follows in
    // memory: they are cleared in the step that holds them.
    const int tail_step = in % V ? in / 32 : -1, tail = in % 32 - 8 * (lane >> 4);
    const auto clear = [&](auto& f) {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = e < tail ? f[e] : 0;
    };

    const bool ragged = out % V != 0;
    // A block's vector stores; ragged columns add some. Between a block's loads
    // and its use: the stores of the kStages - 1 blocks before it (as far as
    // there were any) and the loads of the kStages - 2 blocks after it.
    const int stores = K::kStores * (a.preact.p ? 2 : 1);
    const int step = (int)gridDim.x;
    int before = 0, after = blocks > (int)blockIdx.x ? (blocks - 1 - (int)blockIdx.x) / step : 0, now = 0;
    for (int block = blockIdx.x; block < blocks; block += step) {
        wait_but_for(min(after, K::kStages - 2) * K::kLoads + before * stores);
        before = before < K::kStages - 1 ? before + 1 : before;
        if (after >= K::kStages - 1) load(block + (K::kStages - 1) * step);
        --after;

        const unsigned char* stage = lds + now * K::kStage;
        now = now + 1 < K::kStages ? now + 1 : 0;
        f32x4 acc[2][K::kRowSquares];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int v = 0; v < K::kRowSquares; ++v) acc[u][v] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int s = 0; s < K::kSteps; ++s) {
            if (s >= K::kSteps / 2 && in <= 32 * s) break;   // w is zero there
            typename Frag<T>::type fx[K::kRowSquares];
#pragma unroll
            for (int v = 0; v < K::kRowSquares; ++v) {
                fx[v] = X::k_fragment(stage, (wr * K::kRowSquares + v) * 16, s, lane);
                if (s == tail_step) {
                    if constexpr (sizeof(T) == 4) {
                        clear(fx[v].high);
                        clear(fx[v].middle);
                        clear(fx[v].low);
                    } else {
                        clear(fx[v]);
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int v = 0; v < K::kRowSquares; ++v) acc[u][v] = multiply(fw[u][s], fx[v], acc[u][v]);
        }

        const int64_t first = (int64_t)block * kRows;
        if constexpr (sizeof(T) == 4)
            form_again(
                acc, 0, in,
                [&](int u, int row, int64_t k) {
                    const int64_t n = column0 + 16 * u + row;
                    return n < out ? ((const T*)a.w.p)[n * a.w.stride + k] : 0.0f;
                },
                [&](int v, int row, int64_t k) {
                    const int64_t r = first + (wr * K::kRowSquares + v) * 16 + row;
                    return r < rows ? ((const T*)a.x.p)[r * a.x.stride + k] : 0.0f;
                },
                [](int, int, int) { return true; });
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
            neighbours(acc[0][v], acc[1][v], f);
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] += bias[e];
            const auto store = [&](const __amdgpu_buffer_rsrc_t& buffer, T* p, int64_t stride, int64_t pitch) {
#pragma unroll
                for (int h = 0; h < 8 / V; ++h) {
                    typename K::C::type o;
#pragma unroll
                    for (int e = 0; e < V; ++e) o[e] = (T)f[V * h + e];
                    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, o), buffer,
                                                           (int)((exist >= V * (h + 1) ? 0u : kNowhere) + (uint32_t)r * (uint32_t)pitch +
                                                                 (uint32_t)(at + V * h) * (uint32_t)sizeof(T)),
                                                           0, 0);
                    if (ragged && exist > V * h && exist < V * (h + 1) && r <= held) {
#pragma unroll
                        for (int e = 0; e < V; ++e)
                            if (V * h + e < exist) p[r * stride + V * h + e] = o[e];
                    }
                }
            };
            if (a.preact.p) store(z_buffer, z0, a.preact.stride, z_pitch);
            if (a.activation == kActGelu) activate_all<kActGelu>(f);
            else if (a.activation == kActSilu) activate_all<kActSilu>(f);
            else if (a.activation == kActRelu) activate_all<kActRelu>(f);
            if constexpr (RESIDUAL) {
#pragma unroll
                for (int h = 0; h < 8 / V; ++h) {
                    const auto q = *(const typename K::C::type*)(stage + K::kXBytes + K::R::at(r, (int)(at - c0) / V + h));
#pragma unroll
                    for (int e = 0; e < V; ++e) f[V * h + e] += (float)q[e];
                }
            }
            store(y_buffer, y0, a.y.stride, y_pitch);
        }
    }
}

}  // namespace

// For tests: how far the loads of a block read.
int64_t linear_rows_reach(int64_t left, int64_t cols, int64_t stride, int64_t size) {
    return reach_of(left, (int)cols, (int)stride, (int)size).bytes;
}

// Once a call moves more than the card's last cache holds of it, w in registers
// and few, long waits pay; below, tiles fill the card sooner and their second
// reads of x are from caches. Here and with tiles, us, halves: 262144 x 128 -> 256
// 42 and 52, with gelu, preact and residual 97 and 134; 1e6 x 256 -> 256 so
// 384 and 507; 262144 x 256 -> 128 (201 MB) 44 and 44; 65536 x 128 -> 128 (34 MB)
// 13 and 9. Floats: 182044 x 32 -> 256 (200 MB) 51 and 49, 154202 x 84 -> 256 70
// and 83, with gelu, preact and residual 79996 x 84 -> 256 (260 MB) 60 and 95,
// 76068 x 128 -> 256 67 and 98; the worst, a few in a hundred: 425984 x 32 -> 128
// (260 MB) 63 and 64 but 557056 (340 MB) 90 and 83, 460800 x 128 -> 128 132 and 128.
// Further columns are further workgroups over the same rows: halves 200000 x 128
// -> 1280 179 and 214, -> 4096 413 and 622, 65536 x 256 -> 1280 71 and 71; floats
// 100000 x 128 -> 1024 198 and 206. Past sixteen rows' bytes of them nothing was
// measured, and tiles take it.
// Half of a workgroup's waves have no columns below 128, so those take more:
// halves 262144 x 256 -> 64 (168 MB) 40 and 29, 1e6 x 84 -> 64 (296 MB) 77 and
// 99. Floats multiply six times as long, and the products bound narrow outputs:
// 1e6 x 128 -> 64 197 and 180.
bool linear_forward_by_rows(const LinearForward& a) {
    const bool floats = a.dtype == TGS_DTYPE_FLOAT32;
    const int64_t size = floats ? 4 : 2, most = 512 / size;
    if (a.x.cols > most || a.y.cols > 16 * most) return false;
    const int64_t arrays = 1 + (a.preact.p ? 1 : 0) + (a.residual.p ? 1 : 0);
    const int64_t megabytes = (a.y.rows * (a.x.cols + arrays * a.y.cols) * size) >> 20;
    if (a.y.cols < 128) return !floats && megabytes >= 256;
    return megabytes >= 130;
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
            const int across = (int)((a.y.cols + K::kCols - 1) / K::kCols);
            const int want = 256 * K::kResident / across, down = blocks < want ? blocks : want;   // what the card holds at once
            rows_kernel<T, P, CW, kResidual><<<dim3((unsigned)down, (unsigned)across), kThreads, 0, s>>>(a, blocks);
        };
        const auto by_residual = [&](auto pitch, auto cw) {
            if (a.residual.p) launch(pitch, cw, Constant<1>{});
            else launch(pitch, cw, Constant<0>{});
        };
        const auto by_columns = [&](auto pitch) {
            if constexpr (sizeof(T) == 4) by_residual(pitch, Constant<4>{});
            else if (a.y.cols <= 64) by_residual(pitch, Constant<2>{});
            else if (a.y.cols <= 128) by_residual(pitch, Constant<4>{});
            else by_residual(pitch, Constant<8>{});
        };
        if (a.x.cols <= kMost / 2) by_columns(Constant<256>{});
        else by_columns(Constant<512>{});
    });
}

}  // namespace tgs
