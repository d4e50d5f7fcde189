// Residual addition, root-mean-square norm and int8 activations in one pass (llattn_add_norm_q8).
//
//   v = x + d (fp32; x <- v where there is a d)     r = 1 / sqrt(mean(v^2) + eps)     t = v * gain
//   per group of 128 values:  e = max(max|t| / 127, 1e-30),  code = rint(t / e),  s = e * r,  sum = sum of the codes
//   y = t * r, rounded once to 16 bits (optional)
//
// This is the activation form of the attention epilogue (fragment order, scale and code sum for each group), so llattn_dense_w4a8 reads
// it as it is. The quantiser works on t: r is the same for the whole group and cancels in t / e. So a code waits for its group only, not for
// the row, a row passes through once, and the codes are fixed to the bit by single IEEE operations whatever the order of the row's sum.
//
// A lane holds four neighbouring values of a group (a run of four stays together in fragment order), a warp the group: maximum and code sum
// are one redux instruction each. W warps share a row, group by group in turn; the row's sum of squares is folded lane-wise over a warp's
// groups, by a butterfly over the lanes and over the warps in order, all in fp32.
// Bound by memory from a few thousand rows on (8191 x 2048 with an fp32 addend 37.9 us = 5.8 TB/s), below by the launch and one round trip. The 16-bit copy comes from
// registers where a warp has all of its groups there (rows to 2048 values with 16 or 8 warps a row, to 512 with 4 or 2); beyond that the row and the gain are
// read again, mostly from L2: 8191 x 2048 with a bf16 copy too 46.2 us, its bytes 38.5; 515 x 5120 with an addend and a copy 10.2, its bytes 5.3.
#pragma once

namespace llattn {

struct NormQ8Params {
    float* x;
    const void* d;
    const float* gain;
    int8_t* q;
    float* s;
    int32_t* sum;
    void* y;
    long long ldx, ldd;
    float eps;
    int T, K, y_type;
};

constexpr int NQ_GROUP = 128, NQ_MAX_GROUPS = 256;      // K up to 32,768
constexpr int NQ_NONE = -1;

// Values 4 lane .. 4 lane + 3 of a group of the addend.
template <int DTYPE>
__device__ __forceinline__ float4 norm_load(const void* d, size_t at) {
    if constexpr (DTYPE == LLATTN_F32) return __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(d) + at));
    else {
        const uint2 w = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(d) + at));
        if constexpr (DTYPE == LLATTN_F16) {
            const float2 a = __half22float2(*reinterpret_cast<const half2*>(&w.x)), b = __half22float2(*reinterpret_cast<const half2*>(&w.y));
            return make_float4(a.x, a.y, b.x, b.y);
        } else
            return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u));
    }
}

// Bits of 1.5 * 2^23 + rint(t / e), the quotient rounded as IEEE says. |t / e| is at most 127 and a hair, so the product with the correctly rounded
// reciprocal is within 127.5 * 2^-23 = 1.6e-5 of it, and only a product within 1e-4 of a tie needs the division itself.
__device__ __forceinline__ uint32_t norm_code(float t, float e, float inv) {
    const float a = __fmul_rn(t, inv);
    const float m = __fadd_rn(a, 12582912.f);
    if (!(fabsf(a - __fsub_rn(m, 12582912.f)) < 0.4999f)) return __float_as_uint(__fadd_rn(__fdiv_rn(t, e), 12582912.f));
    return __float_as_uint(m);
}

__device__ __forceinline__ uint2 norm_pack16(const float4& v, int type) {
    uint2 w;
    if (type == LLATTN_F16) {
        const half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
        w.x = *reinterpret_cast<const uint32_t*>(&a); w.y = *reinterpret_cast<const uint32_t*>(&b);
    } else {
        const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
        w.x = *reinterpret_cast<const uint32_t*>(&a); w.y = *reinterpret_cast<const uint32_t*>(&b);
    }
    return w;
}

// W warps share a row, ROWS rows are in a CTA. A warp has the loads of G of its groups in flight.
template <int DTYPE, int W, int ROWS, int G>
__global__ void __launch_bounds__(32 * W * ROWS) add_norm_q8_kernel(const NormQ8Params p) {
    __shared__ float steps[ROWS][NQ_MAX_GROUPS];
    __shared__ float parts[ROWS][W];
    ptx::grid_dependency_wait();               // nothing is read or written before the kernel ahead has completed
    const int lane = threadIdx.x & 31, w = (threadIdx.x >> 5) % W, rr = (threadIdx.x >> 5) / W;
    const int row = blockIdx.x * ROWS + rr, groups = p.K / NQ_GROUP;
    const bool live = row < p.T;
    float* x = p.x + (long long)row * p.ldx + 4 * lane;
    const size_t drow = DTYPE == NQ_NONE ? 0 : size_t(row) * p.ldd + 4 * lane;
    const float* gain = p.gain + 4 * lane;
    const size_t out = size_t(row) * p.K;
    float ss = 0.f;
    float4 v[G];
    if (live) {
#pragma unroll 1
        for (int g0 = w; g0 < groups; g0 += W * G) {
            float4 d[G];
#pragma unroll
            for (int i = 0; i < G; ++i)
                if (g0 + i * W < groups) {
                    v[i] = *reinterpret_cast<const float4*>(x + (g0 + i * W) * NQ_GROUP);
                    if constexpr (DTYPE != NQ_NONE) d[i] = norm_load<DTYPE>(p.d, drow + (g0 + i * W) * NQ_GROUP);
                }
#pragma unroll
            for (int i = 0; i < G; ++i) {
                const int g = g0 + i * W;
                if (g >= groups) break;
                if constexpr (DTYPE != NQ_NONE) {
                    v[i].x += d[i].x; v[i].y += d[i].y; v[i].z += d[i].z; v[i].w += d[i].w;
                    *reinterpret_cast<float4*>(x + g * NQ_GROUP) = v[i];
                }
                ss += v[i].x * v[i].x + v[i].y * v[i].y + v[i].z * v[i].z + v[i].w * v[i].w;
                const float4 gn = __ldg(reinterpret_cast<const float4*>(gain + g * NQ_GROUP));
                v[i] = make_float4(__fmul_rn(v[i].x, gn.x), __fmul_rn(v[i].y, gn.y), __fmul_rn(v[i].z, gn.z), __fmul_rn(v[i].w, gn.w));
                if (p.q) {
                    // of non-negative floats the bits order as the values do, and NaN is above infinity
                    const uint32_t most = max(max(__float_as_uint(fabsf(v[i].x)), __float_as_uint(fabsf(v[i].y))), max(__float_as_uint(fabsf(v[i].z)), __float_as_uint(fabsf(v[i].w))));
                    const float a = __uint_as_float(__reduce_max_sync(0xffffffffu, most));
                    const bool finite = a < INFINITY;
                    const float e = finite ? fmaxf(__fdiv_rn(a, 127.f), 1e-30f) : __uint_as_float(0x7fc00000u);      // else the group's scale is NaN, its codes 0
                    const float inv = __frcp_rn(e);
                    uint32_t word = 0;
                    if (finite) word = __byte_perm(__byte_perm(norm_code(v[i].x, e, inv), norm_code(v[i].y, e, inv), 0x0040),
                                                   __byte_perm(norm_code(v[i].z, e, inv), norm_code(v[i].w, e, inv), 0x0040), 0x5410);
                    const int total = __reduce_add_sync(0xffffffffu, __dp4a(int(word), 0x01010101, 0));
                    *reinterpret_cast<uint32_t*>(p.q + out + frag_pos(g * NQ_GROUP + 4 * lane)) = word;
                    if (lane == 0) {
                        steps[rr][g] = e;
                        p.sum[size_t(row) * groups + g] = total;
                    }
                }
            }
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (lane == 0) parts[rr][w] = ss;
    }
    __syncthreads();
    if (!live) return;
    ss = parts[rr][0];
#pragma unroll
    for (int i = 1; i < W; ++i) ss += parts[rr][i];
    const float r = rsqrtf(ss / float(p.K) + p.eps);
    if (p.q)
        for (int g = 32 * w + lane; g < groups; g += 32 * W) p.s[size_t(row) * groups + g] = __fmul_rn(steps[rr][g], r);
    if (p.y) {
        uint16_t* y = static_cast<uint16_t*>(p.y) + out + 4 * lane;
        auto store = [&](int g, const float4& t) {
            *reinterpret_cast<uint2*>(y + g * NQ_GROUP) = norm_pack16(make_float4(__fmul_rn(t.x, r), __fmul_rn(t.y, r), __fmul_rn(t.z, r), __fmul_rn(t.w, r)), p.y_type);
        };
        if (groups <= W * G) {                 // t is still in the registers
#pragma unroll
            for (int i = 0; i < G; ++i)
                if (w + i * W < groups) store(w + i * W, v[i]);
        } else
            for (int g = w; g < groups; g += W) {      // what this thread has read, or written, above
                const float4 u = *reinterpret_cast<const float4*>(x + g * NQ_GROUP);
                const float4 gn = __ldg(reinterpret_cast<const float4*>(gain + g * NQ_GROUP));
                store(g, make_float4(__fmul_rn(u.x, gn.x), __fmul_rn(u.y, gn.y), __fmul_rn(u.z, gn.z), __fmul_rn(u.w, gn.w)));
            }
    }
}

}  // namespace llattn

namespace {
// How a row is shared. Few rows, or long ones: many warps a row, so that the chip is filled and the chain of a warp short. Many rows: few warps a row, each
// with several groups of loads in flight. In a graph, rows x K, with 16 / 8 / 4 / 2 warps a row: 1 x 2048 2.0 / 2.4 / 3.1 / 6.0 us, 256 x 2048 2.8 / 2.9 /
// 3.6 / 6.9, 512 x 2048 4.7 / 3.9 / 5.4 / 7.9, 515 x 5120 11.2 / 10.1 / 13.4 / 22.9, 1024 x 2048 7.8 / 8.1 / 7.3 / 10.2, 2048 x 2048 13.2 / 13.1 / 12.5 / 13.3,
// 8191 x 2048 46.7 / 41.3 / 39.9 / 37.9, 2000 x 512 9.0 / 7.1 / 4.4 / 3.9, 2048 x 8192 36.2 / 39.2 / 42.4 / 45.1. Between 4096 and 8064 values (fp16 addend): 700 x 4096
// 9.0 / 11.5 / 10.9 / 17.7, 1024 x 4096 12.2 / 13.0 / 12.6 / 18.9, 4096 x 4096 38.5 / 37.9 / 38.1 / 43.6 and without an addend 30.9 / 25.6 / 26.8 / 29.5, 2000 x 6144 28.4 /
// 30.1 / 32.4 / 34.3, 4096 x 8064 69.2 / 69.4 / 72.8 / 89.4: 8 for all of them, best for thousands of rows, up to 3 us behind 16 for a few rows an SM (700 x 7168
// of fp32 14.7 / 17.6).
template <int DTYPE>
cudaError_t launch_norm_q8(const llattn::NormQ8Params& p, int sms, cudaStream_t stream) {
    const int groups = p.K / llattn::NQ_GROUP;
    if (p.T <= 2 * sms || (groups >= 64 && p.T > 4 * sms)) return launch_dependent(llattn::add_norm_q8_kernel<DTYPE, 16, 1, 1>, dim3(p.T), 512, stream, p);
    if (p.T <= 4 * sms || groups >= 32) return launch_dependent(llattn::add_norm_q8_kernel<DTYPE, 8, 1, 2>, dim3(p.T), 256, stream, p);
    if (p.T <= 32 * sms && groups >= 8) return launch_dependent(llattn::add_norm_q8_kernel<DTYPE, 4, 2, 1>, dim3((p.T + 1) / 2), 256, stream, p);
    return launch_dependent(llattn::add_norm_q8_kernel<DTYPE, 2, 4, 2>, dim3((p.T + 3) / 4), 256, stream, p);
}

// Whether two ranges of bytes have one in common.
inline bool overlap(const void* a, unsigned long long na, const void* b, unsigned long long nb) {
    const auto x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return a && b && na && nb && x < y + nb && y < x + na;
}
// The same for two matrices of T rows each, of na and nb bytes, da and db bytes apart: columns of one matrix share no byte though their ranges overlap.
inline bool rows_overlap(const void* a, long long na, long long da, const void* b, long long nb, long long db, long long T) {
    const long long off = (long long)(reinterpret_cast<uintptr_t>(b) - reinterpret_cast<uintptr_t>(a));      // of b's first row from a's
    if (!a || !b || off >= (T - 1) * da + na || -off >= (T - 1) * db + nb) return false;
    // With equal distances the first and the last row of a have all the neighbours that any row has; else each row is looked at.
    for (long long i = 0; i < T; i += da == db ? std::max(T - 1, 1ll) : 1) {
        const long long behind = i * da - off - nb;                // the first row of b that ends behind the beginning of a's row
        const long long j = behind < 0 ? 0 : behind / db + 1;
        if (j < T && off + j * db < i * da + na) return true;
    }
    return false;
}
}  // namespace

extern "C" int llattn_add_norm_q8(float* x, int64_t ldx, const void* delta, int delta_type, int64_t ldd, const float* gain, float eps, int8_t* q,
                                  float* s, int32_t* sum, void* y, int y_type, int T, int K, void* stream) {
    if (!x || !gain) return fail(LLATTN_EINVAL, "add_norm_q8: null pointer");
    if (!q && !y) return fail(LLATTN_EINVAL, "add_norm_q8: no output requested");
    if (q ? (!s || !sum) : (s || sum)) return fail(LLATTN_EINVAL, "add_norm_q8: q, s and sum go together");
    if (T < 0 || T > 1 << 24) return fail(LLATTN_EINVAL, "add_norm_q8: T = %d", T);
    if (K <= 0 || K % llattn::NQ_GROUP || K > llattn::NQ_GROUP * llattn::NQ_MAX_GROUPS) return fail(LLATTN_EINVAL, "add_norm_q8: K = %d (a multiple of 128 up to 32768)", K);
    const int64_t far = int64_t(1) << 32;
    if (ldx < K || ldx % 4 || ldx > far || (delta && (ldd < K || ldd % 4 || ldd > far)))
        return fail(LLATTN_EINVAL, "add_norm_q8: rows %lld and %lld apart (at least K, multiples of 4)", (long long)ldx, (long long)ldd);
    if (delta && (delta_type < LLATTN_F32 || delta_type > LLATTN_BF16)) return fail(LLATTN_EINVAL, "add_norm_q8: delta_type = %d", delta_type);
    if (y && y_type != LLATTN_F16 && y_type != LLATTN_BF16) return fail(LLATTN_EINVAL, "add_norm_q8: y_type = %d", y_type);
    if (!(eps >= 0.f) || !(eps < INFINITY)) return fail(LLATTN_EINVAL, "add_norm_q8: eps = %g", double(eps));
    if (!aligned16(x) || !aligned16(delta) || !aligned16(gain) || !aligned16(q) || !aligned16(y))
        return fail(LLATTN_EINVAL, "add_norm_q8: x, delta, gain, q and y must be 16-byte aligned");
    if (reinterpret_cast<uintptr_t>(s) % 4 || reinterpret_cast<uintptr_t>(sum) % 4) return fail(LLATTN_EINVAL, "add_norm_q8: s and sum must be 4-byte aligned");
    if (T == 0) return LLATTN_OK;
    const long long esize = delta_type == LLATTN_F32 ? 4 : 2;
    // (x and delta may be columns of one matrix, so it is their rows that count)
    struct { const void* p; unsigned long long n; bool out; } const m[] = {
        {x, (unsigned long long)((T - 1) * ldx + K) * 4, delta != nullptr}, {delta, delta ? (unsigned long long)((T - 1) * ldd + K) * esize : 0, false},
        {gain, (unsigned long long)K * 4, false}, {q, (unsigned long long)T * K, true}, {s, (unsigned long long)T * K / 32, true},
        {sum, (unsigned long long)T * K / 32, true}, {y, (unsigned long long)T * K * 2, true}};
    for (int i = 0; i < 7; ++i)
        for (int j = 0; j < i; ++j)
            if ((m[i].out || m[j].out) && overlap(m[i].p, m[i].n, m[j].p, m[j].n) && (i != 1 || rows_overlap(x, 4ll * K, 4 * ldx, delta, esize * K, esize * ldd, T)))
                return fail(LLATTN_EINVAL, "add_norm_q8: an output overlaps another argument");
    int dev = 0, sms = 0;
    CU(cudaGetDevice(&dev));
    CU(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    const llattn::NormQ8Params p{x, delta, gain, q, s, sum, y, ldx, ldd, eps, T, K, y_type};
    if (!delta) CU(launch_norm_q8<llattn::NQ_NONE>(p, sms, as_stream(stream)));
    else if (delta_type == LLATTN_F32) CU(launch_norm_q8<LLATTN_F32>(p, sms, as_stream(stream)));
    else if (delta_type == LLATTN_F16) CU(launch_norm_q8<LLATTN_F16>(p, sms, as_stream(stream)));
    else CU(launch_norm_q8<LLATTN_BF16>(p, sms, as_stream(stream)));
    return LLATTN_OK;
}
