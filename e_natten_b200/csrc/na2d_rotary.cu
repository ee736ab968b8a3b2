// Rotary positions on queries and keys (include/na2d.h).
//
//   (a, b) -> (a cos - b sin, b cos + a sin) for each pair of the first `dims` channels; the others are copied.
//
// Bound by memory: q and k are read and written once, in one launch.  A thread has two vectors of one token (in the half layout the
// ones that its pairs lie in) and takes them through several heads, so that the table's cosines and sines, as many bytes as the
// vectors' own in 32 bits, are read once for all of them.  Measured: 4 x 4 heads x 256^2 x 128, bf16, forward and backward in 385 us, 88 % of
// the copy bandwidth; 64 single tokens 8 us, the host's time of the call.
#include <cuda_runtime.h>

#include <algorithm>

#include "../../include/na2d.h"
#include "na2d_host.h"
#include "na2d_launch.h"
#include "na2d_ptx.cuh"
#include "na2d_vec.cuh"

namespace {

using na2d_vec::Vec;

constexpr int kThreads = 256;

struct Side {               // q or k
    const void* in;
    void* out;
    long long b, n, t;      // of the input; the output is dense
    int heads;
};

struct Rotary {
    Side side[2];
    int B, T, C, half;      // half: pairs
    int turned, items;      // vector pairs of a token that turn, and in all
    int step;               // heads of a thread
    int interleaved, index_64;
    float sign;             // of the sines
    const float2* table;    // (rows, half)
    long long rows;
    const void* index;
};

// Vectors of a token that item i has: [0] and [1] of `at`, in vectors of N channels; the second may be missing (-1).
template <int N>
__device__ __forceinline__ void vectors_of(const Rotary& r, int i, int (&at)[2]) {
    if (i < r.turned && !r.interleaved) {                    // channels i N ... and half + i N ...
        at[0] = i;
        at[1] = r.half / N + i;
        return;
    }
    const int first = i < r.turned ? 0 : 2 * r.half / N, end = i < r.turned ? 2 * r.half / N : r.C / N;
    at[0] = first + 2 * (i < r.turned ? i : i - r.turned);
    at[1] = at[0] + 1 < end ? at[0] + 1 : -1;
}

template <typename T, int N>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const Rotary r) {
    na2d_ptx::after_previous_grid();
    na2d_ptx::next_grid_may_start();
    const long long id = (long long)blockIdx.x * kThreads + threadIdx.x;
    const long long token = id / r.items;
    if (token >= (long long)r.B * r.T) return;
    const int item = (int)(id - token * r.items);
    const int b = (int)(token / r.T), t = (int)(token - (long long)b * r.T);
    int at[2];
    vectors_of<N>(r, item, at);
    const bool turn = item < r.turned, both = at[1] >= 0;

    // cosine and sine of the N pairs (half layout: pair i of both vectors) or of N / 2 pairs of each vector
    float2 cs[N];
    if (turn) {
        const long long row = !r.index ? t
                              : r.index_64 ? static_cast<const long long*>(r.index)[token]
                                           : (long long)static_cast<const int*>(r.index)[token];
        const bool known = row >= 0 && row < r.rows;
        const float2* src = r.table + (known ? row * r.half : 0) + item * N;
        const int pairs = r.interleaved && !both ? N / 2 : N;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            cs[i] = i < pairs ? __ldg(src + i) : make_float2(1.f, 0.f);
            cs[i].y *= r.sign;
            if (!known) cs[i] = make_float2(__int_as_float(0x7fc00000), 0.f);
        }
    }
    // heads of q, then of k
    const int heads = r.side[0].heads + r.side[1].heads;
    const int h0 = blockIdx.y * r.step, h1 = min(heads, h0 + r.step);
#pragma unroll 4
    for (int h = h0; h < h1; ++h) {
        const bool second = h >= r.side[0].heads;
        const Side &q = r.side[0], &k = r.side[1];
        const T* src = second ? static_cast<const T*>(k.in) + b * k.b + (h - q.heads) * k.n + t * k.t
                              : static_cast<const T*>(q.in) + b * q.b + h * q.n + t * q.t;
        T* dst = second ? static_cast<T*>(k.out) + (((long long)b * k.heads + h - q.heads) * r.T + t) * r.C
                        : static_cast<T*>(q.out) + (((long long)b * q.heads + h) * r.T + t) * r.C;
        Vec<T, N> x, y;
        x.load(src + at[0] * N);
        if (both) y.load(src + at[1] * N);
        if (turn) {
            float f[N], e[N];
            x.widened(f);
            if (both) y.widened(e);
            if (!r.interleaved) {
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const float u = f[i], v = e[i];
                    f[i] = fmaf(u, cs[i].x, -(v * cs[i].y));
                    e[i] = fmaf(v, cs[i].x, u * cs[i].y);
                }
            } else if constexpr (N > 1) {
#pragma unroll
                for (int i = 0; i < N / 2; ++i) {
                    const float u = f[2 * i], v = f[2 * i + 1];
                    f[2 * i] = fmaf(u, cs[i].x, -(v * cs[i].y));
                    f[2 * i + 1] = fmaf(v, cs[i].x, u * cs[i].y);
                }
                if (both) {
#pragma unroll
                    for (int i = 0; i < N / 2; ++i) {
                        const float u = e[2 * i], v = e[2 * i + 1];
                        e[2 * i] = fmaf(u, cs[N / 2 + i].x, -(v * cs[N / 2 + i].y));
                        e[2 * i + 1] = fmaf(v, cs[N / 2 + i].x, u * cs[N / 2 + i].y);
                    }
                }
            } else {                                         // the two vectors are one pair
                const float u = f[0], v = e[0];
                f[0] = fmaf(u, cs[0].x, -(v * cs[0].y));
                e[0] = fmaf(v, cs[0].x, u * cs[0].y);
            }
            x.round(f);
            if (both) y.round(e);
        }
        x.store(dst + at[0] * N);
        if (both) y.store(dst + at[1] * N);
    }
}

__global__ void __launch_bounds__(kThreads)
rotary_table_kernel(const double* __restrict__ positions, const double* __restrict__ frequencies, float2* __restrict__ table, long long P,
                    int axes, int pairs, double magnitude) {
    const long long id = (long long)blockIdx.x * kThreads + threadIdx.x;
    const int width = axes * pairs;
    if (id >= P * width) return;
    const long long p = id / width;
    const int i = (int)(id - p * width);
    double s, c;
    sincos(positions[p * axes + i / pairs] * frequencies[i], &s, &c);
    table[id] = make_float2((float)(magnitude * c), (float)(magnitude * s));
}

// Channels of a vector: 16 bytes' where everything is a multiple of them, else 4 bytes', else one.
int vector_of(const Rotary& r, int esize) {
    auto fits = [&](int v) {
        const int bytes = v * esize;
        bool ok = r.C % v == 0 && (r.interleaved ? 2 * r.half : r.half) % v == 0;
        for (const Side& s : r.side)
            ok = ok && (!s.heads || (reinterpret_cast<uintptr_t>(s.in) % bytes == 0 && reinterpret_cast<uintptr_t>(s.out) % bytes == 0 &&
                                     s.b % v == 0 && s.n % v == 0 && s.t % v == 0));
        return ok;
    };
    const int full = 16 / esize, small = 4 / esize;
    return fits(full) ? full : small > 1 && fits(small) ? small : 1;
}

template <typename T, int N>
int launch_rotary(Rotary r, int sms, cudaStream_t st) {
    r.turned = r.interleaved && N > 1 ? (2 * r.half / N + 1) / 2 : r.half / N;
    r.items = r.turned + ((r.C - 2 * r.half) / N + 1) / 2;
    const long long threads = (long long)r.B * r.T * r.items;
    const long long blocks = (threads + kThreads - 1) / kThreads;
    if (blocks > 0x7fffffffLL) return NA2D_ERR_TOO_LARGE;
    // heads of a thread: 8, fewer where that would leave SMs without four blocks
    const int heads = r.side[0].heads + r.side[1].heads;
    r.step = (int)std::max(1LL, std::min(8LL, blocks * heads / (4 * sms)));
    const long long parts = (heads + r.step - 1) / r.step;
    if (parts > 65535) return NA2D_ERR_TOO_LARGE;
    const cudaError_t e = na2d_launch::launch(true, rotary_kernel<T, N>, dim3((unsigned)blocks, (unsigned)parts), kThreads, 0, st, r);
    if (e != cudaSuccess) return na2d_host::cuda_fail(e, "rotary launch");
    na2d_host::count_launches(1);
    return NA2D_OK;
}

template <typename T>
int by_vector(const Rotary& r, int sms, cudaStream_t st) {
    constexpr int kFull = 16 / (int)sizeof(T), kSmall = 4 / (int)sizeof(T);
    const int v = vector_of(r, sizeof(T));
    return v == kFull ? launch_rotary<T, kFull>(r, sms, st) : v == kSmall ? launch_rotary<T, kSmall>(r, sms, st) : launch_rotary<T, 1>(r, sms, st);
}

}  // namespace

extern "C" {

int na2d_rotary(const na2d_rotary_args* a) {
    if (!a || a->struct_size < sizeof(na2d_rotary_args)) return NA2D_ERR_BAD_ARG;
    if (!a->q.ptr || !a->out_q || !a->table || (a->k.ptr && !a->out_k)) return NA2D_ERR_BAD_ARG;
    if (a->B <= 0 || a->N <= 0 || a->T <= 0 || a->C <= 0 || (a->k.ptr && a->Nk <= 0)) return NA2D_ERR_BAD_ARG;
    if (a->dims <= 0 || a->dims % 2 != 0 || a->dims > a->C || a->table_rows <= 0) return NA2D_ERR_BAD_ARG;
    if (!a->index && a->table_rows < a->T) return NA2D_ERR_BAD_ARG;
    if (a->dtype != NA2D_F32 && a->dtype != NA2D_BF16 && a->dtype != NA2D_F16) return NA2D_ERR_UNSUPPORTED;
    if ((reinterpret_cast<uintptr_t>(a->table) & 7u) != 0) return NA2D_ERR_BAD_ARG;
    Rotary r{};
    auto side = [&](const na2d_heads& x, void* out, int heads) {
        const na2d_host::HeadStrides s = na2d_host::head_strides(x, a->B, heads, a->T, a->C);
        return Side{x.ptr, out, s.b, s.n, s.t, heads};
    };
    r.side[0] = side(a->q, a->out_q, a->N);
    if (a->k.ptr) r.side[1] = side(a->k, a->out_k, a->Nk);
    r.B = a->B;
    r.T = a->T;
    r.C = a->C;
    r.half = a->dims / 2;
    r.interleaved = a->interleaved != 0;
    r.index_64 = a->index_64 != 0;
    r.sign = a->inverse ? -1.f : 1.f;
    r.table = reinterpret_cast<const float2*>(a->table);
    r.rows = a->table_rows;
    r.index = a->index;
    return na2d_host::on_device(a->device, [&]() -> int {
        const cudaStream_t st = (cudaStream_t)a->stream;
        const int sms = na2d_host::sm_count(a->device);
        return a->dtype == NA2D_F32    ? by_vector<float>(r, sms, st)
               : a->dtype == NA2D_BF16 ? by_vector<__nv_bfloat16>(r, sms, st)
                                       : by_vector<__half>(r, sms, st);
    });
}

int na2d_rotary_table(const double* positions, const double* frequencies, int64_t P, int axes, int pairs, double magnitude,
                      float* table, int device, void* stream) {
    if (!positions || !frequencies || !table || P <= 0 || axes <= 0 || pairs <= 0) return NA2D_ERR_BAD_ARG;
    if (axes > (1 << 15) || pairs > (1 << 15) || P > (1ll << 31)) return NA2D_ERR_TOO_LARGE;
    const long long values = P * axes * pairs, blocks = (values + kThreads - 1) / kThreads;
    if (blocks > 0x7fffffffLL) return NA2D_ERR_TOO_LARGE;
    return na2d_host::on_device(device, [&]() -> int {
        rotary_table_kernel<<<(unsigned)blocks, kThreads, 0, (cudaStream_t)stream>>>(positions, frequencies, reinterpret_cast<float2*>(table), P,
                                                                                       axes, pairs, magnitude);
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return na2d_host::cuda_fail(e, "rotary table launch");
        na2d_host::count_launches(1);
        return NA2D_OK;
    });
}

}  // extern "C"
