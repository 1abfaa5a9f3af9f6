// The global norm of a list of gradients and their clipping:
//   norm = scale sqrt(sum over all tensors of g^2),   out = g * scale * min(1, max_norm / (norm + 1e-6)).
//
// Two launches over the whole list, whose addresses and sizes travel as kernel parameters.  (1) square_sums_kernel: every CTA adds up the
// squares of the chunks that are its own by index, in fp64, and leaves one number.  (2) clip_kernel: every CTA adds up these numbers
// in the same order -- all have the same norm, whichever CTA ran first -- and multiplies its chunks, the last ones first: what
// the first launch read last is still in L2.  Where the factor is 1 and the gradients stay where they are it ends there.
// No atomics, nothing to clear, no CTA waits for another.  Bound by HBM: the gradients are read twice, less what L2 keeps, and written once.
//
// fp64: an SM has 64 fp64 FMAs a clock, and HBM brings it 6 fp32 or 12 16-bit elements; squares of all fp32 numbers are finite and
// not 0 there, so that a norm neither overflows nor vanishes before the result is rounded to fp32.
#include "common.cuh"

namespace sfb {
namespace gn {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kMostChunk = 16384, kLeastChunk = 2048;      // elements: a CTA's unit, shorter where the list is
constexpr uint32_t kMost = 768;                      // tensors per launch (kernel parameters: 32764 bytes)
constexpr uint32_t kCtasPerSm = 4;
// Shared memory that a CTA asks for and does not use: no SM then takes more than four.  Launched behind each other's back, the second launch's CTAs
// went eight at a time to the first SMs that had room, and half of the SMs had none (clipping 334 M elements 468 -> 834 us).
constexpr size_t kRoom = 46 * 1024;
static_assert(kCtasPerSm * (kRoom + 1024) <= 228 * 1024 && (kCtasPerSm + 1) * (kRoom + 1024) > 228 * 1024, "four CTAs per SM, not five");

struct Entry {
    const void *in;
    void *out;
    uint64_t n;
};
template <uint32_t M> struct List {
    Entry t[M];
    uint32_t first[M + 1];                           // chunk at which tensor i begins; first[count]: all chunks
    uint8_t types[M];                                // in | out << 4
    uint32_t count, chunk;
};

template <int DT> __device__ __forceinline__ float widen(const typename Elem<DT>::type &v)
{
    return Elem<DT>::load(&v, 0);
}
// 16 bytes of elements
template <int DT> struct Vec {
    static constexpr int N = DT == SFB_F32 ? 4 : 8;
    static __device__ __forceinline__ void decode(float (&v)[N], const uint4 &u)
    {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (DT == SFB_F32) {
                v[i] = __uint_as_float(w[i]);
            } else if constexpr (DT == SFB_BF16) {
                v[2 * i] = __uint_as_float(w[i] << 16);
                v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            } else {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
                v[2 * i] = f.x;
                v[2 * i + 1] = f.y;
            }
        }
    }
};

// the tensor that chunk c belongs to
template <uint32_t M> __device__ __forceinline__ uint32_t find(const List<M> &l, uint32_t c)
{
    uint32_t lo = 0, hi = l.count;                   // first[lo] <= c < first[hi]
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (l.first[mid] <= c) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Sum of the squares of a piece.  fp32: each in fp64.  16 bits: a product of two is exact in fp32 and four of them are added there (three
// roundings, 2^-24 each of at most the sum), which leaves a quarter of the conversions and fp64 additions: all in fp64, 334 M fp16
// elements took 182 us.  bf16 squares that leave fp32's range, or come near its end, are made in fp64.
template <int DT> __device__ __forceinline__ void add_squares(double &s0, double &s1, const uint4 &u)
{
    float v[Vec<DT>::N];
    Vec<DT>::decode(v, u);
    if constexpr (DT == SFB_F32) {
        s0 = fma((double)v[0], (double)v[0], s0);
        s1 = fma((double)v[1], (double)v[1], s1);
        s0 = fma((double)v[2], (double)v[2], s0);
        s1 = fma((double)v[3], (double)v[3], s1);
    } else {
        const uint32_t any[2] = {(u.x | u.y) & 0x7fff7fffu, (u.z | u.w) & 0x7fff7fffu};
        double *s[2] = {&s0, &s1};
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const float *x = v + 4 * h;
            const float p = fmaf(x[0], x[0], x[1] * x[1]) + fmaf(x[2], x[2], x[3] * x[3]);
            if (DT == SFB_F16 || (p > 1e-30f && p < 1e37f)) {
                *s[h] += (double)p;
            } else if (any[h]) {
#pragma unroll
                for (int j = 0; j < 4; j++) *s[h] = fma((double)x[j], (double)x[j], *s[h]);
            }
        }
    }
}
constexpr int kAhead = 8;                            // 16-byte loads of a thread on their way
template <int DT> __device__ __forceinline__ double chunk_squares(const void *in, uint64_t begin, uint64_t end)
{
    constexpr int N = Vec<DT>::N;
    const typename Elem<DT>::type *p = (const typename Elem<DT>::type *)in;
    double s0 = 0.0, s1 = 0.0;
    // up to the first 16-byte boundary, whole pieces, the rest
    const uint64_t lead = ((16 - ((uintptr_t)(p + begin) & 15)) & 15) / sizeof(*p), body = min(end, begin + lead), tail = body + (end - body) / N * N;
    const uint32_t pieces = (uint32_t)((tail - body) / N);
    if (begin + threadIdx.x < body) {
        const double v = widen<DT>(p[begin + threadIdx.x]);
        s0 = v * v;
    }
    const uint4 *q = (const uint4 *)(p + body);
    uint32_t i = threadIdx.x;
    for (; i + (kAhead - 1) * kThreads < pieces; i += kAhead * kThreads) {
        uint4 u[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; k++) u[k] = __ldg(q + i + k * kThreads);
#pragma unroll
        for (int k = 0; k < kAhead; k++) add_squares<DT>(s0, s1, u[k]);
    }
    for (; i < pieces; i += kThreads) add_squares<DT>(s0, s1, __ldg(q + i));
    if (tail + threadIdx.x < end) {
        const double v = widen<DT>(p[tail + threadIdx.x]);
        s1 = fma(v, v, s1);
    }
    return s0 + s1;
}

__device__ __forceinline__ double block_sum(double v)
{
    __shared__ double part[kThreads / 32];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0;
#pragma unroll
    for (uint32_t w = 0; w < kThreads / 32; w++) v += part[w];
    return v;
}

template <uint32_t M>
__global__ void __launch_bounds__(kThreads) square_sums_kernel(const __grid_constant__ List<M> l, double *sums)
{
    grid_dependency_wait();
    grid_launch_dependents();
    const uint32_t chunks = l.first[l.count];
    double s = 0.0;
    for (uint32_t c = blockIdx.x; c < chunks; c += gridDim.x) {
        const uint32_t i = find(l, c);
        const uint64_t begin = (uint64_t)(c - l.first[i]) * l.chunk, end = min(l.t[i].n, begin + l.chunk);
        const int t = l.types[i] & 15;
        s += t == SFB_F32 ? chunk_squares<SFB_F32>(l.t[i].in, begin, end) : t == SFB_BF16 ? chunk_squares<SFB_BF16>(l.t[i].in, begin, end) : chunk_squares<SFB_F16>(l.t[i].in, begin, end);
    }
    s = block_sum(s);
    if (threadIdx.x == 0) sums[blockIdx.x] = s;
}

template <int GT> __device__ __forceinline__ void put(void *out, uint64_t i, float v)
{
    if constexpr (GT == SFB_F32) ((float *)out)[i] = v;
    else if constexpr (GT == SFB_BF16) ((__nv_bfloat16 *)out)[i] = __float2bfloat16_rn(v);
    else ((__half *)out)[i] = __float2half_rn(v);
}
// wide: 32-byte pieces of fp32 results at their boundaries, one store (as two, each covers half of every sector)
template <int GT, int N> __device__ __forceinline__ void put_vec(void *out, uint64_t i, const float (&v)[N], bool wide)
{
    if constexpr (GT == SFB_F32) {
        if constexpr (N == 8) {
            if (wide) {
                asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"((float *)out + i), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]),
                             "f"(v[6]), "f"(v[7])
                             : "memory");
                return;
            }
        }
#pragma unroll
        for (int j = 0; j < N; j += 4) __stcs((float4 *)((float *)out + i + j), make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]));
    } else {
        static_assert(N == 8, "16 bytes");
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if constexpr (GT == SFB_BF16) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
                w[j] = *reinterpret_cast<const uint32_t *>(&h);
            } else {
                const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
                w[j] = *reinterpret_cast<const uint32_t *>(&h);
            }
        }
        __stcs((uint4 *)((uint16_t *)out + i), make_uint4(w[0], w[1], w[2], w[3]));
    }
}
template <int DT, int GT>
__device__ __forceinline__ void chunk_scale(const void *in, void *out, uint64_t begin, uint64_t end, float factor)
{
    constexpr int N = Vec<DT>::N, S = sizeof(typename Elem<DT>::type), G = GT == SFB_F32 ? 4 : 2;
    const typename Elem<DT>::type *p = (const typename Elem<DT>::type *)in;
    // whole pieces of 16 bytes where both sides have their boundaries at the same elements
    const uint64_t lead = ((16 - ((uintptr_t)(p + begin) & 15)) & 15) / S;
    const bool vec = (((uintptr_t)out + (begin + lead) * G) & 15) == 0;
    if (vec) {
        const uint64_t body = min(end, begin + lead), tail = body + (end - body) / N * N;
        const uint32_t pieces = (uint32_t)((tail - body) / N);
        if (begin + threadIdx.x < body) put<GT>(out, begin + threadIdx.x, widen<DT>(p[begin + threadIdx.x]) * factor);
        if (tail + threadIdx.x < end) put<GT>(out, tail + threadIdx.x, widen<DT>(p[tail + threadIdx.x]) * factor);
        const uint4 *q = (const uint4 *)(p + body);
        const bool wide = (((uintptr_t)out + body * G) & 31) == 0;
        auto scale_piece = [&](uint32_t i, const uint4 &u) {
            float v[N];
            Vec<DT>::decode(v, u);
#pragma unroll
            for (int j = 0; j < N; j++) v[j] *= factor;
            put_vec<GT>(out, body + (uint64_t)i * N, v, wide);
        };
        // the results may lie where the gradients do: what is on its way together has to be asked for before the first of it is written
        uint32_t i = threadIdx.x;
        for (; i + 3 * kThreads < pieces; i += 4 * kThreads) {
            uint4 u[4];
#pragma unroll
            for (int k = 0; k < 4; k++) u[k] = q[i + k * kThreads];
#pragma unroll
            for (int k = 0; k < 4; k++) scale_piece(i + k * kThreads, u[k]);
        }
        for (; i < pieces; i += kThreads) scale_piece(i, q[i]);
    } else {
        uint64_t i = begin + threadIdx.x;
        for (; i + (kAhead - 1) * kThreads < end; i += kAhead * kThreads) {
            float v[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; k++) v[k] = widen<DT>(p[i + k * kThreads]) * factor;
#pragma unroll
            for (int k = 0; k < kAhead; k++) put<GT>(out, i + k * kThreads, v[k]);
        }
        for (; i < end; i += kThreads) put<GT>(out, i, widen<DT>(p[i]) * factor);
    }
}

// 334 M fp16 gradients into fp32: 345 us, 2.0 GB at 5.8 TB/s (with one load at a time and two stores per 32 bytes 352; eight loads 355).
// max_norm: infinity where only the norm is wanted.  parts: how many numbers the launches before left.
template <uint32_t M>
__global__ void __launch_bounds__(kThreads) clip_kernel(const __grid_constant__ List<M> l, const double *sums, uint32_t parts, float *norm_out, float max_norm, float scale,
                                                       int in_place)
{
    grid_dependency_wait();
    grid_launch_dependents();
    double s = 0.0;
    for (uint32_t i = threadIdx.x; i < parts; i += kThreads) s += sums[i];
    s = block_sum(s);
    const double norm = sqrt(s) * (double)scale;
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
    const float shown = (float)norm;
    if (!(shown <= 3.402823466e38f)) return;         // infinite or NaN: nothing is written
    const float factor = (float)((double)scale * fmin(1.0, (double)max_norm / (norm + 1e-6)));
    if (in_place && factor == 1.f) return;
    const uint32_t chunks = l.first[l.count];
    for (uint32_t k = blockIdx.x; k < chunks; k += gridDim.x) {
        const uint32_t c = chunks - 1 - k, i = find(l, c);
        const uint64_t begin = (uint64_t)(c - l.first[i]) * l.chunk, end = min(l.t[i].n, begin + l.chunk);
        const void *in = l.t[i].in;
        void *out = l.t[i].out;
        switch (l.types[i]) {
            case SFB_F32 | SFB_F32 << 4: chunk_scale<SFB_F32, SFB_F32>(in, out, begin, end, factor); break;
            case SFB_BF16 | SFB_F32 << 4: chunk_scale<SFB_BF16, SFB_F32>(in, out, begin, end, factor); break;
            case SFB_F16 | SFB_F32 << 4: chunk_scale<SFB_F16, SFB_F32>(in, out, begin, end, factor); break;
            case SFB_BF16 | SFB_BF16 << 4: chunk_scale<SFB_BF16, SFB_BF16>(in, out, begin, end, factor); break;
            default: chunk_scale<SFB_F16, SFB_F16>(in, out, begin, end, factor); break;
        }
    }
}

static uint32_t most_ctas(int sms) { return kCtasPerSm * (uint32_t)sms; }

template <uint32_t M>
static void fill(List<M> &l, uint32_t from, uint32_t count, const void *const *grads, void *const *out, const uint64_t *numel, const int32_t *dtypes, const int32_t *out_dtypes)
{
    uint32_t chunks = 0;
    for (uint32_t i = 0; i < count; i++) {
        const uint32_t k = from + i;
        l.t[i] = {grads[k], out ? out[k] : (void *)grads[k], numel[k]};
        l.first[i] = chunks;
        l.types[i] = (uint8_t)(dtypes[k] | (out ? out_dtypes[k] : dtypes[k]) << 4);
        chunks += (uint32_t)((numel[k] + l.chunk - 1) / l.chunk);
    }
    l.first[count] = chunks;
    l.count = count;
}

template <uint32_t M>
static int run(cudaStream_t s, uint32_t count, const void *const *grads, void *const *out, const uint64_t *numel, const int32_t *dtypes, const int32_t *out_dtypes, float max_norm,
               float scale, float *norm, double *sums, bool write)
{
    const int sms = device_sm_count(current_device());
    if (sms <= 0) return fail("sfb_clip_grad_norm: cannot query the device");
    uint32_t parts = 0;
    List<M> l;
    uint64_t all = 0;
    for (uint32_t i = 0; i < count; i++) all += numel[i];
    l.chunk = kMostChunk;                            // a list that gives the SMs few chunks is cut finer
    while (l.chunk > kLeastChunk && all / l.chunk < 4ull * most_ctas(sms)) l.chunk /= 2;
    for (uint32_t from = 0; from < count || from == 0; from += M) {
        fill<M>(l, from, count - from < M ? count - from : M, grads, out, numel, dtypes, out_dtypes);
        const uint32_t chunks = l.first[l.count], ctas = chunks < most_ctas(sms) ? (chunks ? chunks : 1) : most_ctas(sms);
        launch_overlapped(square_sums_kernel<M>, dim3(ctas), dim3(kThreads), kRoom, s, l, sums + parts);
        parts += ctas;
    }
    for (uint32_t from = 0; from < count || from == 0; from += M) {
        if (count > M) fill<M>(l, from, count - from < M ? count - from : M, grads, out, numel, dtypes, out_dtypes);
        const uint32_t chunks = write ? l.first[l.count] : 0, ctas = chunks < most_ctas(sms) ? (chunks ? chunks : 1) : most_ctas(sms);
        if (!write) l.count = 0, l.first[0] = 0;
        launch_overlapped(clip_kernel<M>, dim3(ctas), dim3(kThreads), kRoom, s, l, sums, parts, from ? nullptr : norm, max_norm, scale, (int)(out == nullptr));
        if (!write) break;
    }
    return check_launch("sfb_clip_grad_norm");
}

}  // namespace gn
}  // namespace sfb

using namespace sfb;

extern "C" uint64_t sfb_clip_grad_norm_workspace(uint32_t count)
{
    const int sms = device_sm_count(current_device());
    return (uint64_t)(count / gn::kMost + 1) * gn::most_ctas(sms > 0 ? sms : 256) * sizeof(double);
}

static int grad_norm_common(const char *who, sfb_stream_t stream, uint32_t count, const void *const *grads, void *const *out, const uint64_t *numel,
                            const int32_t *dtypes, const int32_t *out_dtypes, float max_norm, float scale, float *norm, void *workspace, bool write)
{
    SFB_REQUIRE(norm && workspace && (count == 0 || (grads && numel && dtypes)) && (!out || out_dtypes), "%s: NULL pointer", who);
    SFB_REQUIRE(((uintptr_t)workspace & 7) == 0, "%s: the workspace must be 8-byte aligned", who);
    SFB_REQUIRE(max_norm >= 0.f, "%s: max_norm must not be negative or NaN", who);
    SFB_REQUIRE(scale > 0.f && scale <= 3.402823466e38f, "%s: scale must be positive and finite", who);
    uint64_t chunks = 0;
    for (uint32_t i = 0; i < count; i++) {
        SFB_REQUIRE(valid_dtype(dtypes[i]) && (!out || out_dtypes[i] == dtypes[i] || out_dtypes[i] == SFB_F32), "%s: tensor %u: unknown dtype, or a result neither fp32 nor of its type", who, i);
        SFB_REQUIRE(numel[i] == 0 || (grads[i] && (!out || out[i])), "%s: tensor %u: NULL pointer", who, i);
        SFB_REQUIRE(((uintptr_t)grads[i] & (elem_size(dtypes[i]) - 1)) == 0 && (!out || ((uintptr_t)out[i] & (elem_size(out_dtypes[i]) - 1)) == 0),
                    "%s: tensor %u is not aligned to its elements", who, i);
        chunks += numel[i] / gn::kLeastChunk + 1;
        SFB_REQUIRE(chunks < (1ull << 31), "%s: too many elements", who);
    }
    cudaStream_t s = as_stream(stream);
    if (count <= 64) return gn::run<64>(s, count, grads, out, numel, dtypes, out_dtypes, max_norm, scale, norm, (double *)workspace, write);
    return gn::run<gn::kMost>(s, count, grads, out, numel, dtypes, out_dtypes, max_norm, scale, norm, (double *)workspace, write);
}

extern "C" int sfb_grad_norm(sfb_stream_t stream, uint32_t count, const void *const *grads, const uint64_t *numel, const int32_t *dtypes, float scale,
                             float *norm, void *workspace)
{
    return grad_norm_common("sfb_grad_norm", stream, count, grads, nullptr, numel, dtypes, nullptr, INFINITY, scale, norm, workspace, false);
}

extern "C" int sfb_clip_grad_norm(sfb_stream_t stream, uint32_t count, const void *const *grads, void *const *out, const uint64_t *numel,
                                  const int32_t *dtypes, const int32_t *out_dtypes, float max_norm, float scale, float *norm, void *workspace)
{
    return grad_norm_common("sfb_clip_grad_norm", stream, count, grads, out, numel, dtypes, out_dtypes, max_norm, scale, norm, workspace, true);
}
