// Rows of logits, read 16 bytes at a time: what the kernels of logits.cu share.
//
// A row is cut into WINDOWS of 16 bytes at 16-byte boundaries of memory, whatever element it starts with: 8 elements of a
// 16-bit type, 4 of fp32.  Windows that lie inside the row are one load; the first and the last may hold elements of
// neighbouring rows (or padding), which are never read: they come as -inf, a probability of 0.
#pragma once
#include "common.cuh"
#include "attn.cuh"

namespace sfb {
namespace lg {

constexpr uint32_t kNoWindow = 0xffffffffu;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kFar = -2000.f;       // an exponent (base 2) whose power is 0 and whose product with it is, too: keeps 0 * -inf out of sums

template <int DT> struct Win {
    static constexpr uint32_t kElems = DT == SFB_F32 ? 4 : 8;
    static constexpr uint32_t kSize = DT == SFB_F32 ? 4 : 2;
    static constexpr uint32_t kInf = DT == SFB_F32 ? 0xff800000u : DT == SFB_BF16 ? 0xff80u : 0xfc00u;      // -inf
};

__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// two fp32 values as one operand of the packed instructions, which do both at the cost of one
typedef unsigned long long Pair;
__device__ __forceinline__ Pair pair(float a, float b)
{
    Pair p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(a), "f"(b));
    return p;
}
__device__ __forceinline__ void halves(Pair p, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p)); }
__device__ __forceinline__ Pair add2(Pair a, Pair b)
{
    Pair p;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(p) : "l"(a), "l"(b));
    return p;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b)
{
    Pair p;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(p) : "l"(a), "l"(b));
    return p;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c)
{
    Pair p;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(p) : "l"(a), "l"(b), "l"(c));
    return p;
}
// the larger one, NaN if either is NaN
__device__ __forceinline__ float max_nan(float a, float b)
{
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
__device__ __forceinline__ float neg_inf() { return __uint_as_float(0xff800000u); }

// The windows of one row: n elements from x on.
template <int DT> struct Row {
    const uint4 *base;          // the first window
    uint32_t head, end;         // the row's elements are the positions [head, end) of its windows
    __device__ __forceinline__ Row(const void *x, uint32_t n)
    {
        const uintptr_t a = (uintptr_t)x;
        base = (const uint4 *)(a & ~(uintptr_t)15);
        head = (uint32_t)(a & 15) / Win<DT>::kSize;
        end = head + n;
    }
    __device__ __forceinline__ uint32_t windows() const { return (end + Win<DT>::kElems - 1) / Win<DT>::kElems; }
    // windows [first_whole, first_whole + whole_count) are inside the row; besides them there are at most two
    __device__ __forceinline__ uint32_t first_whole() const { return head ? 1 : 0; }
    __device__ __forceinline__ uint32_t whole_count() const
    {
        const uint32_t b = first_whole(), e = end / Win<DT>::kElems;
        return e > b ? e - b : 0;
    }
    __device__ __forceinline__ uint32_t front() const { return head ? 0u : kNoWindow; }
    __device__ __forceinline__ uint32_t back() const
    {
        const uint32_t w = end / Win<DT>::kElems;
        return end % Win<DT>::kElems && !(w == 0 && head) ? w : kNoWindow;
    }
    __device__ __forceinline__ bool whole(uint32_t w) const { return w * Win<DT>::kElems >= head && (w + 1) * Win<DT>::kElems <= end; }
};

// A window that is not inside the row as a whole, element by element.
template <int DT> __device__ __noinline__ uint4 edge_window(const uint4 *base, uint32_t head, uint32_t end, uint32_t w)
{
    uint32_t v[4];
#pragma unroll
    for (uint32_t j = 0; j < 4; j++) {
        const uint32_t pos = w * Win<DT>::kElems + j * (Win<DT>::kElems / 4);
        if (DT == SFB_F32) {
            v[j] = pos >= head && pos < end ? ((const uint32_t *)base)[pos] : Win<DT>::kInf;
        } else {
            const uint32_t lo = pos >= head && pos < end ? ((const uint16_t *)base)[pos] : Win<DT>::kInf;
            const uint32_t hi = pos + 1 >= head && pos + 1 < end ? ((const uint16_t *)base)[pos + 1] : Win<DT>::kInf;
            v[j] = lo | hi << 16;
        }
    }
    return make_uint4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ uint4 load16(const uint4 *p)
{
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
template <int DT> __device__ __forceinline__ uint4 no_elements()
{
    const uint32_t none = DT == SFB_F32 ? Win<DT>::kInf : Win<DT>::kInf << 16 | Win<DT>::kInf;
    return make_uint4(none, none, none, none);
}
template <int DT> __device__ __forceinline__ uint4 load_window(const Row<DT> &r, uint32_t w)
{
    if (r.whole(w)) return load16(r.base + w);
    if (w * Win<DT>::kElems >= r.end) return no_elements<DT>();
    return edge_window<DT>(r.base, r.head, r.end, w);
}

// element e of a word of a window (two elements of a 16-bit type, one of fp32)
template <int DT> __device__ __forceinline__ float lower(uint32_t v)
{
    if (DT == SFB_F32) return __uint_as_float(v);
    if (DT == SFB_BF16) return __uint_as_float(v << 16);
    return __half2float(__ushort_as_half((unsigned short)(v & 0xffff)));
}
template <int DT> __device__ __forceinline__ float upper(uint32_t v)
{
    if (DT == SFB_BF16) return __uint_as_float(v & 0xffff0000u);
    return __half2float(__ushort_as_half((unsigned short)(v >> 16)));
}
template <int DT> __device__ __forceinline__ void unpack(const uint4 &v, float (&x)[Win<DT>::kElems])
{
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; j++) {
        if (DT == SFB_F32) {
            x[j] = lower<DT>(u[j]);
        } else {
            x[(2 * j) % Win<DT>::kElems] = lower<DT>(u[j]);
            x[(2 * j + 1) % Win<DT>::kElems] = upper<DT>(u[j]);
        }
    }
}
template <int DT> __device__ __forceinline__ uint32_t max_word(uint32_t a, uint32_t b)
{
    uint32_t y;
    if (DT == SFB_F32) asm("max.NaN.f32 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
    else if (DT == SFB_BF16) asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
    else asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
    return y;
}
// largest element of N windows, NaN if there is one
template <int DT, int N> __device__ __forceinline__ float max_windows(const uint4 (&v)[N])
{
    uint32_t m = max_word<DT>(max_word<DT>(v[0].x, v[0].y), max_word<DT>(v[0].z, v[0].w));
#pragma unroll
    for (int u = 1; u < N; u++) m = max_word<DT>(m, max_word<DT>(max_word<DT>(v[u].x, v[u].y), max_word<DT>(v[u].z, v[u].w)));
    return DT == SFB_F32 ? lower<DT>(m) : max_nan(lower<DT>(m), upper<DT>(m));
}

template <int DT> __device__ __forceinline__ float load_element(const void *x, uint32_t i)
{
    if (DT == SFB_F32) return ((const float *)x)[i];
    if (DT == SFB_BF16) return from_bhalf_bits(((const uint16_t *)x)[i]);
    return __half2float(((const __half *)x)[i]);
}
// results are rounded to the nearest, ties to even: half a unit in the last place
template <int DT> __device__ __forceinline__ void store_element(void *x, uint32_t i, float v)
{
    if (DT == SFB_F32) ((float *)x)[i] = v;
    else if (DT == SFB_BF16) ((__nv_bfloat16 *)x)[i] = __float2bfloat16_rn(v);
    else ((__half *)x)[i] = __float2half_rn(v);
}
template <int DT> __device__ __forceinline__ uint4 pack(const float (&x)[Win<DT>::kElems])
{
    uint32_t u[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        if (DT == SFB_F32) u[j] = __float_as_uint(x[j]);
        else if (DT == SFB_BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(u[j]) : "f"(x[(2 * j + 1) % Win<DT>::kElems]), "f"(x[(2 * j) % Win<DT>::kElems]));
        else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(u[j]) : "f"(x[(2 * j + 1) % Win<DT>::kElems]), "f"(x[(2 * j) % Win<DT>::kElems]));
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
}

// Sum of 2^(s2 (x - r)) and of its terms times their exponents, beside a reference r that is one of the values seen.  The
// reference moves only when a value outgrows it by 2^40: the sums stay far inside fp32, and no pass for the maximum is needed.
struct Sums {
    float r, lim, s, e;
    __device__ __forceinline__ Sums() : r(neg_inf()), lim(neg_inf()), s(0.f), e(0.f) {}
    // before values whose largest is m; false: all of them are -inf and so is everything before them
    __device__ __forceinline__ bool prepare(float m, float s2, float gap)
    {
        if (!(m <= lim)) {
            if (m > neg_inf()) {
                if (r > neg_inf()) rescale(m, s2);
                r = m;
                lim = m + gap;
            } else {
                s = m;                  // a NaN among them
            }
        }
        return r > neg_inf();
    }
    __device__ __forceinline__ void rescale(float m, float s2)
    {
        const float d = fmaxf(s2 * (r - m), kFar), f = ex2(d);
        e = f * fmaf(d, s, e);
        s *= f;
    }
    // to the reference m, at least the largest value seen
    __device__ __forceinline__ void move_to(float m, float s2)
    {
        if (r > neg_inf()) rescale(m, s2);
        r = m;
    }
};

}  // namespace lg
}  // namespace sfb
