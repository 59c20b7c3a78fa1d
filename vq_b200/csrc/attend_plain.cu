// attend_plain.cu -- attention over a cache of 8-bit codes on the CUDA cores, which VQB_NO_TENSOR=1 selects.
//
//   y_i = sum_j e^(S_ij - m_i) s_v v_j / sum_j e^(S_ij - m_i),  S_ij = scale (x_i . k_j) s_k,  over the tokens j that row i sees
//
// A warp for each row and query head.  s_v enters with its exponent in the power: values of pages whose scales are far apart keep their weights.
#include <algorithm>

#include "cache.cuh"
#include "cuda_device.hpp"

namespace vqb {

namespace {

constexpr int THREADS = 256;

__global__ void __launch_bounds__(THREADS) attend_plain_kernel(const Attend P)
{
    cache_is_there();
    const Cache &c = P.cache;
    const int lane = threadIdx.x % 32, heads = (int)c.heads * P.group, width = (int)c.width, padded = (int)c.padded;
    const size_t at = ((size_t)blockIdx.x * THREADS + threadIdx.x) / 32;
    if (at >= (size_t)P.seq.n * heads) return;
    const int r = (int)(at / heads), qh = (int)(at % heads), h = qh / P.group;
    const int i = sequence_of(P.seq, r, 1, 0);
    const Span span(P.seq, i);
    const size_t yo = (size_t)r * P.y.ld + (size_t)qh * P.y.head_ld, xo = (size_t)r * P.queries.ld + (size_t)qh * P.queries.head_ld;
    if (r < span.row || r >= span.row + span.count) {
        if (P.zero_rest)
            for (int d = lane; d < width; d += 32) put_value(P.y, yo + d, 0.0f);
        return;
    }
    const int position = span.first + r - span.row, last = min(position, span.keys - 1), begin = P.window ? max(max(position, 0) - P.window + 1, 0) : 0;
    float x[8], y[8] = {};
#pragma unroll
    for (int d = 0; d < 8; ++d) x[d] = lane + 32 * d < width ? value_at(P.queries, xo + lane + 32 * d) : 0.0f;
    float m = -INFINITY, l = 0.0f, top = -INFINITY; // top: the largest of S + the exponent of s_v, what the values' weights are relative to
    for (int j = 0; j <= last; ++j) {
        if (j >= P.sinks && j < begin) {
            j = begin - 1;
            continue;
        }
        const int p = page_of(P.seq, c.pages, i, j / CACHE_PAGE);
        if (p < 0) continue;
        const size_t part = (size_t)p * c.heads + h;
        const uint8_t *codes = c.codes + part * 2 * CACHE_PAGE * padded, *v = codes + CACHE_PAGE * padded + j % CACHE_PAGE;
        const int t = j % CACHE_PAGE;
        const float ks = c.scales[2 * part], vs = c.scales[2 * part + 1];
        float s = 0.0f;
#pragma unroll
        for (int d = 0; d < 8; ++d)
            if (32 * d < padded) s = fmaf(x[d], (float)((int)codes[key_at(padded, t, lane + 32 * d)] - 128), s);
#pragma unroll
        for (int o = 16; o; o /= 2) s += __shfl_xor_sync(~0u, s, o);
        s *= ks * P.scale;
        const float up = s > m || s != s ? s : m;
        l = l * (m == -INFINITY ? 0.0f : expf(m - up)) + expf(s - up), m = up;
        if (vs == 0.0f) continue;
        int e = 0;
        const float f = vs == vs ? frexpf(vs, &e) : vs, se = s + e * 0.69314718f, higher = se > top || se != se ? se : top;
        const float old = top == -INFINITY ? 0.0f : expf(top - higher), w = expf(se - higher) * f;
        top = higher;
#pragma unroll
        for (int d = 0; d < 8; ++d)
            if (32 * d < padded) y[d] = fmaf(w, (float)((int)v[(lane + 32 * d) * CACHE_PAGE] - 128), y[d] * old);
    }
#pragma unroll
    for (int d = 0; d < 8; ++d)
        if (lane + 32 * d < width) put_value(P.y, yo + lane + 32 * d, l == 0.0f || top == -INFINITY ? l == l ? 0.0f : l : y[d] / l * expf(top - m));
}

} // namespace

void launch_attend_plain(CudaDevice &dev, const Attend &a)
{
    const size_t warps = (size_t)a.seq.n * a.cache.heads * a.group;
    KernelScope ks(dev, "attend_plain");
    launch_following(attend_plain_kernel, dim3((unsigned)((warps + THREADS / 32 - 1) / (THREADS / 32))), dim3(THREADS), 0, dev.stream(), a);
    dev.count_launch();
}

} // namespace vqb
