// Rows into microscaled form and back, and the residual sum with its RMS norm straight into that form (see microscaled.cuh for the layout).
// All three read every input once and write every output once; what bounds them is memory.
#include "microscaled.cuh"

namespace lb {

constexpr int kMicroscaleThreads = 256;

// Division of numbers below 2^31 by one that the host knows: with l = ceil(log2 d) and m = ceil(2^(31 + l) / d), n / d = n m >> (31 + l), exact for those n
// (m d exceeds 2^(31 + l) by less than d <= 2^l).
struct Divisor {
    unsigned divisor, multiplier, shift;
    __device__ __forceinline__ unsigned quotient(unsigned n) const { return divisor == 1 ? n : __umulhi(n, multiplier) >> shift; }
};
inline Divisor divisor_of(unsigned d) {
    unsigned l = 0;
    while ((1ull << l) < d) ++l;
    return {d, d == 1 ? 0u : static_cast<unsigned>(((1ull << (31 + l)) + d - 1) / d), l - 1};
}

// Pieces of 128 columns under one word of scales, `chunks` of them a row, LANES lanes to each; a block takes ROUNDS rounds of them.  (There are fewer than
// 2^31: the rows would not fit the GPU.)
struct Piece {
    int row, chunk;
    bool exists;
};
template <int LANES, int ROUNDS>
__device__ __forceinline__ Piece piece_of(int u, unsigned total, const Divisor& chunks) {
    const unsigned piece = (blockIdx.x * ROUNDS + u) * (kMicroscaleThreads / LANES) + threadIdx.x / LANES;
    const unsigned row = chunks.quotient(piece);
    return {static_cast<int>(row), static_cast<int>(piece - row * chunks.divisor), piece < total};
}
template <int LANES, int ROUNDS>
dim3 microscale_grid(unsigned pieces) {
    constexpr unsigned per_block = kMicroscaleThreads / LANES * ROUNDS;
    return dim3((pieces + per_block - 1) / per_block);
}

// How many columns of x a lane takes at a time and how often, by the type.  Of bfloat16 sixteen, two loads of 16 bytes: what is done once a lane, places and scales, is
// then half of what it is with eight, and instructions bound that (16,384 x 2,048 to 8 bits: 15.9 us, 6.4 TB/s, and 19.7 with eight).  Of float32, which memory bounds,
// eight and once (25.7 us, 6.6 TB/s; four times 27.8).
template <typename T>
struct MicroscaleShape {
    static constexpr int kCount = sizeof(T) == 2 ? 16 : 8, kLanes = 128 / kCount, kRounds = sizeof(T) == 2 ? 2 : 1;
};
// The same of the values' kernel: eight columns, four times of bfloat16 (14.9 us, 6.8 TB/s; once 19.9), once of float32 (32.0 us; four times 36.4), without the launch behind it.
template <typename T>
constexpr int kValuesRounds = sizeof(T) == 2 ? 4 : 1;

// codes and scales of x [rows, width]
template <typename T, int BITS, bool VECTOR>
__global__ void __launch_bounds__(kMicroscaleThreads)
microscale_kernel(const T* __restrict__ x, unsigned char* __restrict__ codes, unsigned char* __restrict__ scales, int width, unsigned total, Divisor chunks) {
    constexpr int kCount = MicroscaleShape<T>::kCount, kLanes = MicroscaleShape<T>::kLanes, kRounds = MicroscaleShape<T>::kRounds;
    wait_for_previous_kernel();
    allow_next_kernel();
    const int column = threadIdx.x % kLanes * kCount;
    Piece piece[kRounds];
    float v[kRounds][kCount];
#pragma unroll
    for (int u = 0; u < kRounds; ++u) {
        piece[u] = piece_of<kLanes, kRounds>(u, total, chunks);
        // a piece that does not exist counts as one past its row's width: zeros
        const T* row = x + static_cast<size_t>(piece[u].row) * width;
        const int first = piece[u].exists ? piece[u].chunk * 128 + column : width;
        load_eight<VECTOR>(row, first, width, v[u]);
        if constexpr (kCount == 16) load_eight<VECTOR, 8>(row, first + 8, width, v[u]);
    }
#pragma unroll
    for (int u = 0; u < kRounds; ++u) {
        uint32_t code[kCount * BITS / 32];
        const uint32_t word = quantise<BITS>(v[u], code);
        if (!piece[u].exists) continue;
        store_codes(codes + ((static_cast<size_t>(piece[u].row) * chunks.divisor + piece[u].chunk) * 128 + column) * BITS / 8, code);
        if (column == 0) *reinterpret_cast<uint32_t*>(scales + scale_word(piece[u].row, piece[u].chunk, chunks.divisor)) = word;
    }
}

// The values [rows, width] that codes and scales stand for, rounded once to the output's type (e4m3 and e2m1 elements times their scale are exact in
// bfloat16 down to its subnormals).
template <typename T, int BITS, bool VECTOR>
__global__ void __launch_bounds__(kMicroscaleThreads)
microscaled_values_kernel(const unsigned char* __restrict__ codes, const unsigned char* __restrict__ scales, T* __restrict__ out, int width, unsigned total, Divisor chunks) {
    wait_for_previous_kernel();
    constexpr int kRounds = kValuesRounds<T>;
    const int column = (threadIdx.x & 15) * 8;
    Piece piece[kRounds];
    uint2 code[kRounds];
    int byte[kRounds];
#pragma unroll
    for (int u = 0; u < kRounds; ++u) {
        piece[u] = piece_of<16, kRounds>(u, total, chunks);
        if (!piece[u].exists) continue;
        const size_t at = (static_cast<size_t>(piece[u].row) * chunks.divisor + piece[u].chunk) * 128 + column;
        if constexpr (BITS == 8) code[u] = *reinterpret_cast<const uint2*>(codes + at);
        else code[u].x = *reinterpret_cast<const uint32_t*>(codes + at / 2);
        byte[u] = scales[scale_word(piece[u].row, piece[u].chunk, chunks.divisor) + column / 32];
    }
#pragma unroll
    for (int u = 0; u < kRounds; ++u) {
        if (!piece[u].exists) continue;
        const float scale = scale_value(byte[u]);
        float v[8];
        unpack_eight<BITS>(code[u], v);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= scale;
        store_eight<VECTOR>(out + static_cast<size_t>(piece[u].row) * width, piece[u].chunk * 128 + column, width, v);
    }
}

// Nothing, launched the ordinary way behind the values: they may be a weight, and a bfloat16 product asks for its first tiles of W before it waits for the kernel in front of it.
// It starts when this has ended, and this when the values are written; so does every product after it.  (A kernel that merely does not let its successor start early ends
// before its writes are seen to.)  Costs 1 us of the device's time.
__global__ void values_are_written_kernel() {}

// s = x + delta; sum_out = s; y = s * rsqrt(mean(s^2) + eps) * (weight + offset), microscaled from 32 bits.  A block per row, GROUPS pieces of eight
// columns a thread, which stay in registers between the sum of squares and the norm.  sum_out may be x: an element is read and written by one thread.
template <typename TD, int BITS, int GROUPS, bool VECTOR>
__global__ void __launch_bounds__(GROUPS == 4 ? 1024 : 256)
rmsnorm_microscaled_kernel(const float* x, const TD* __restrict__ delta, float* sum_out, const float* __restrict__ weight, float offset, float eps,
                           unsigned char* __restrict__ codes, unsigned char* __restrict__ scales, int width, int chunks) {
    __shared__ float scratch[33];
    wait_for_previous_kernel();
    allow_next_kernel();
    const int row = blockIdx.x;
    const size_t base = static_cast<size_t>(row) * width;
    float v[GROUPS][8];
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) load_eight<VECTOR>(x + base, (threadIdx.x + g * blockDim.x) * 8, width, v[g]);
    if (delta != nullptr) {
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
            float d[8];
            load_eight<VECTOR>(delta + base, (threadIdx.x + g * blockDim.x) * 8, width, d);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[g][i] += d[i];
        }
    }
    float squares = 0.0f;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
        if (sum_out != nullptr) store_eight<VECTOR>(sum_out + base, (threadIdx.x + g * blockDim.x) * 8, width, v[g]);
#pragma unroll
        for (int i = 0; i < 8; ++i) squares += v[g][i] * v[g][i];
    }
    const float factor = rsqrtf(block_sum(squares, scratch) / static_cast<float>(width) + eps);
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
        const int column = (threadIdx.x + g * blockDim.x) * 8;
        float w[8];
        load_eight<VECTOR>(weight, column, width, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = column + i < width ? v[g][i] * factor * (w[i] + offset) : 0.0f;
        uint32_t code[BITS / 4];
        const uint32_t word = quantise<BITS>(w, code);
        if (column >= chunks * 128) continue;
        store_codes(codes + (static_cast<size_t>(row) * chunks * 128 + column) * BITS / 8, code);
        if ((column & 127) == 0) *reinterpret_cast<uint32_t*>(scales + scale_word(row, column >> 7, chunks)) = word;
    }
}

template <typename T>
bool rows_are_aligned(const T* rows, int width) {
    return width % 8 == 0 && (reinterpret_cast<uintptr_t>(rows) & 15) == 0;
}

template <typename T, int BITS>
cudaError_t launch_microscale(const T* x, unsigned char* codes, unsigned char* scales, int rows, int width, cudaStream_t stream) {
    const int chunks = (width + 127) / 128;
    auto kernel = rows_are_aligned(x, width) ? microscale_kernel<T, BITS, true> : microscale_kernel<T, BITS, false>;
    return launch_overlapped(kernel, microscale_grid<MicroscaleShape<T>::kLanes, MicroscaleShape<T>::kRounds>(static_cast<unsigned>(rows) * chunks), dim3(kMicroscaleThreads), 0, stream, x, codes, scales, width,
                             static_cast<unsigned>(rows) * chunks, divisor_of(chunks));
}

template <typename T, int BITS>
cudaError_t launch_values(const unsigned char* codes, const unsigned char* scales, T* out, int rows, int width, cudaStream_t stream) {
    const int chunks = (width + 127) / 128;
    auto kernel = rows_are_aligned(out, width) ? microscaled_values_kernel<T, BITS, true> : microscaled_values_kernel<T, BITS, false>;
    const cudaError_t error = launch_overlapped(kernel, microscale_grid<16, kValuesRounds<T>>(static_cast<unsigned>(rows) * chunks), dim3(kMicroscaleThreads), 0, stream, codes, scales, out,
                                                width, static_cast<unsigned>(rows) * chunks, divisor_of(chunks));
    if (error != cudaSuccess) return error;
    values_are_written_kernel<<<1, 32, 0, stream>>>();
    return cudaGetLastError();
}

template <typename TD, int BITS, int GROUPS>
cudaError_t launch_norm_groups(const float* x, const TD* delta, float* sum_out, const float* weight, float offset, float eps, unsigned char* codes,
                               unsigned char* scales, int rows, int width, cudaStream_t stream) {
    const int chunks = (width + 127) / 128, groups = chunks * 16;
    const int threads = ((groups + GROUPS - 1) / GROUPS + 31) / 32 * 32;
    const bool aligned = rows_are_aligned(x, width) && rows_are_aligned(delta, width) && rows_are_aligned(sum_out, width) && rows_are_aligned(weight, width);
    auto kernel = aligned ? rmsnorm_microscaled_kernel<TD, BITS, GROUPS, true> : rmsnorm_microscaled_kernel<TD, BITS, GROUPS, false>;
    return launch_overlapped(kernel, dim3(rows), dim3(threads), 0, stream, x, delta, sum_out, weight, offset, eps, codes, scales, width, chunks);
}

constexpr int kNormLargestWidth = 32768;   // 1024 threads of four pieces of eight columns

template <typename TD, int BITS>
cudaError_t launch_norm(const float* x, const TD* delta, float* sum_out, const float* weight, float offset, float eps, unsigned char* codes,
                        unsigned char* scales, int rows, int width, cudaStream_t stream) {
    if (width <= 2048) return launch_norm_groups<TD, BITS, 1>(x, delta, sum_out, weight, offset, eps, codes, scales, rows, width, stream);
    if (width <= 4096) return launch_norm_groups<TD, BITS, 2>(x, delta, sum_out, weight, offset, eps, codes, scales, rows, width, stream);
    return launch_norm_groups<TD, BITS, 4>(x, delta, sum_out, weight, offset, eps, codes, scales, rows, width, stream);
}

}  // namespace lb

extern "C" {

// Return codes: 0, a CUDA error, -1 for an element type, -2 for sizes that the kernels do not take.

int lb_microscale(const void* x, void* codes, void* scales, int rows, int width, int bits, int dtype, cudaStream_t stream) {
    if (rows < 0 || width < 1 || (bits != 4 && bits != 8) || static_cast<long long>(rows) * ((width + 127ll) / 128) >= 1ll << 31) return -2;
    if (rows == 0) return 0;
    unsigned char *c = static_cast<unsigned char*>(codes), *s = static_cast<unsigned char*>(scales);
    LB_DISPATCH_DTYPE(dtype, {
        const T* source = static_cast<const T*>(x);
        return static_cast<int>(bits == 8 ? lb::launch_microscale<T, 8>(source, c, s, rows, width, stream) : lb::launch_microscale<T, 4>(source, c, s, rows, width, stream));
    })
}

int lb_microscaled_values(const void* codes, const void* scales, void* out, int rows, int width, int bits, int dtype, cudaStream_t stream) {
    if (rows < 0 || width < 1 || (bits != 4 && bits != 8) || static_cast<long long>(rows) * ((width + 127ll) / 128) >= 1ll << 31) return -2;
    if (rows == 0) return 0;
    const unsigned char *c = static_cast<const unsigned char*>(codes), *s = static_cast<const unsigned char*>(scales);
    LB_DISPATCH_DTYPE(dtype, {
        T* destination = static_cast<T*>(out);
        return static_cast<int>(bits == 8 ? lb::launch_values<T, 8>(c, s, destination, rows, width, stream) : lb::launch_values<T, 4>(c, s, destination, rows, width, stream));
    })
}

// delta (may be null) has the type `dtype`; sum_out may be null, or x.
int lb_rmsnorm_microscaled(const float* x, const void* delta, float* sum_out, const float* weight, float offset, float eps, void* codes, void* scales, int rows,
                           int width, int bits, int dtype, cudaStream_t stream) {
    if (rows < 0 || width < 1 || width > lb::kNormLargestWidth || (bits != 4 && bits != 8)) return -2;
    if (rows == 0) return 0;
    unsigned char *c = static_cast<unsigned char*>(codes), *s = static_cast<unsigned char*>(scales);
    LB_DISPATCH_DTYPE(dtype, {
        const T* d = static_cast<const T*>(delta);
        return static_cast<int>(bits == 8 ? lb::launch_norm<T, 8>(x, d, sum_out, weight, offset, eps, c, s, rows, width, stream)
                                          : lb::launch_norm<T, 4>(x, d, sum_out, weight, offset, eps, c, s, rows, width, stream));
    })
}

}  // extern "C"
