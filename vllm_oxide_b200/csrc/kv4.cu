// Writing and reading the 4-bit cache (layout and numbers: kv4.cuh): append with the rotary positions applied on the way, read back,
// and attention in 32-bit arithmetic for every type and size. The tensor-core kernels of single tokens and of portions are in kv4_decode.cu
// and kv4_prefill.cu.
#include "kv4.cuh"
VOB_PDL_SWITCH(kv4)

namespace {
using namespace vob_kv4;

// ---------------------------------------------------------------------------------------------
// Append. For every token: q and k rotated by the angles position * inv_freq (float32, as everywhere in this package), k (as
// rotated, not rounded to the activations' type first) and v quantised and written to the token's slot.
//
// A code is a decision: a key within a rounding of the border of two codes would land on either side, a whole step apart. So the
// rotation of k is taken in 64 bits (sine and cosine once per token and pair, shared by all heads) and rounded to 32 bits
// once; scale, minimum and codes are then fixed operations in 32 bits with one rounding each (no contraction into FMAs).
//
// One block per token (and per share of its vectors, where there are few tokens), eight warps that walk over its H + 2 G
// vectors. LANES lanes hold a vector: unit u is the numbers 2u, 2u + 1 and their partners D/2 + 2u, D/2 + 2u + 1, that is one byte of codes in each half.
// Bound: memory (reads q, k, v once, writes q and 136 of 512 bytes per key and value at D = 128).
// ---------------------------------------------------------------------------------------------
constexpr int APPEND_THREADS = 256;

template <typename T> __device__ __forceinline__ float2 load2(const T* p, bool vec);
template <> __device__ __forceinline__ float2 load2<float>(const float* p, bool vec) {
    if (vec) return *reinterpret_cast<const float2*>(p);
    return make_float2(p[0], p[1]);
}
template <> __device__ __forceinline__ float2 load2<__nv_bfloat16>(const __nv_bfloat16* p, bool vec) {
    if (vec) return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(p));
    return make_float2(__bfloat162float(p[0]), __bfloat162float(p[1]));
}
template <typename T> __device__ __forceinline__ void store2(T* p, float2 v, bool vec);
template <> __device__ __forceinline__ void store2<float>(float* p, float2 v, bool vec) {
    if (vec) *reinterpret_cast<float2*>(p) = v;
    else { p[0] = v.x; p[1] = v.y; }
}
template <> __device__ __forceinline__ void store2<__nv_bfloat16>(__nv_bfloat16* p, float2 v, bool vec) {
    if (vec) *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(v.x, v.y);
    else { p[0] = __float2bfloat16_rn(v.x); p[1] = __float2bfloat16_rn(v.y); }
}

__device__ __forceinline__ int code_of(float x, float m, float s) {
    const float n = rintf(__fdiv_rn(__fsub_rn(x, m), s));
    return (int)fminf(fmaxf(n, 0.f), 15.f);               // NaN (s is NaN): 0
}

// LANES lanes quantise one vector: lane `l` of them holds units l, l + LANES, ...: x[2i] the low pair, x[2i + 1] the high pair. Called by
// whole warps (the reductions need every lane); vectors that are not kept have `store` false.
template <int LANES, int UNITS>
__device__ __forceinline__ void quantise_store(const float2 (&x)[2 * UNITS], int l, int hd, bool store, unsigned char* codes, int lane8,
                                               uint32_t* params) {
    const int units = hd >> 2;
    float lo = INFINITY, hi = -INFINITY;
    bool fin = true;
#pragma unroll
    for (int i = 0; i < UNITS; ++i)
        if (l + i * LANES < units) {
            const float2 a = x[2 * i], b = x[2 * i + 1];
            lo = fminf(lo, fminf(fminf(a.x, a.y), fminf(b.x, b.y)));
            hi = fmaxf(hi, fmaxf(fmaxf(a.x, a.y), fmaxf(b.x, b.y)));
            fin = fin && isfinite(a.x) && isfinite(a.y) && isfinite(b.x) && isfinite(b.y);
        }
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        fin = __shfl_xor_sync(0xffffffffu, (int)fin, o) && fin;
    }
    if (!store) return;
    const float fifteenth = 0.06666667014360428f;
    __nv_bfloat16 sb = __float2bfloat16_rn(__fsub_rn(__fmul_rn(hi, fifteenth), __fmul_rn(lo, fifteenth)));
    __nv_bfloat16 mb = __float2bfloat16_rn(lo);
    if (!fin) sb = mb = __float2bfloat16_rn(NAN);          // a vector with a number that is not finite is kept as NaN
    const float s = __bfloat162float(sb), m = __bfloat162float(mb);
    const int last = 16 * chunks(hd);                      // bytes of codes, the rest of the last chunk included
#pragma unroll
    for (int i = 0; i < UNITS; ++i) {
        const int u = l + i * LANES;
        if (u < units) {
            const float2 a = x[2 * i], b = x[2 * i + 1];
            int na = 0, nb = 0;
            if (s != 0.f) {
                na = code_of(a.x, m, s) | code_of(a.y, m, s) << 4;
                nb = code_of(b.x, m, s) | code_of(b.y, m, s) << 4;
            }
            const int ub = u + units;
            codes[(u >> 4) * 128 + lane8 * 16 + (u & 15)] = (unsigned char)na;
            codes[(ub >> 4) * 128 + lane8 * 16 + (ub & 15)] = (unsigned char)nb;
        }
    }
    const int tail = 2 * units + l;                        // the rest of the last chunk: at most 8 bytes (head sizes are multiples of 16)
    if (tail < last) codes[(tail >> 4) * 128 + lane8 * 16 + (tail & 15)] = 0;
    if (l == 0) *params = (uint32_t)__bfloat16_as_ushort(sb) | (uint32_t)__bfloat16_as_ushort(mb) << 16;
}

template <typename T, int LANES, int UNITS>
__global__ void __launch_bounds__(APPEND_THREADS)
kv4_append_kernel(const T* q, long long q_stride, T* q_out, long long qo_stride, const T* __restrict__ k, long long k_stride,
                  const T* __restrict__ v, long long v_stride, const int* __restrict__ positions, const int* __restrict__ slots,
                  const float* __restrict__ inv_freq, unsigned char* __restrict__ cache, long long num_slots, int H, int G, int hd,
                  int page_size, bool vec) {
    __shared__ double2 turn[128];                          // cosine and sine of the token's angles
    pdl_launch_dependents();
    pdl_wait(30);
    const int t = blockIdx.x, half = hd >> 1;
    if (inv_freq) {
        const float pos = (float)positions[t];
        for (int i = threadIdx.x; i < half; i += APPEND_THREADS) {
            const float theta = pos * inv_freq[i];
            double s, c;
            sincospi((double)theta * 0.31830988618379067154, &s, &c);
            turn[i] = make_double2(c, s);
        }
    } else {
        for (int i = threadIdx.x; i < half; i += APPEND_THREADS) turn[i] = make_double2(1.0, 0.0);
    }
    __syncthreads();
    const int slot = slots ? slots[t] : -1;
    const bool keep = slot >= 0 && slot < num_slots;
    const int page = keep ? slot / page_size : 0, off = keep ? slot - page * page_size : 0;
    const int C = chunks(hd), width = token_bytes(hd), units = hd >> 2;
    constexpr int PER_WARP = 32 / LANES;                   // vectors a warp works on side by side
    const int l = threadIdx.x % LANES;
    const int first = (blockIdx.y * (APPEND_THREADS / 32) + (threadIdx.x >> 5)) * PER_WARP + (threadIdx.x & 31) / LANES;
    const int step = gridDim.y * (APPEND_THREADS / 32) * PER_WARP;
    const int vectors = H + 2 * G;
    // every lane of a warp takes part in the reductions: the loop runs as long as one of its vectors is there
    for (int e0 = first - (threadIdx.x & 31) / LANES; e0 < vectors; e0 += step) {
        const int e = e0 + (threadIdx.x & 31) / LANES;
        const bool is_q = e < H, is_k = !is_q && e < H + G, there = e < vectors;
        const int head = is_q ? e : is_k ? e - H : e - H - G;
        const T* src = is_q ? q + (size_t)t * q_stride : is_k ? k + (size_t)t * k_stride : v + (size_t)t * v_stride;
        src += (size_t)head * hd;
        float2 x[2 * UNITS];
#pragma unroll
        for (int i = 0; i < UNITS; ++i) {
            const int u = l + i * LANES;
            x[2 * i] = x[2 * i + 1] = make_float2(0.f, 0.f);
            if (there && u < units) {
                float2 a = load2(src + 2 * u, vec), b = load2(src + half + 2 * u, vec);
                if (is_q || is_k) {
                    const double2 t0 = turn[2 * u], t1 = turn[2 * u + 1];
                    const double ax = a.x, ay = a.y, bx = b.x, by = b.y;
                    a = make_float2((float)(ax * t0.x - bx * t0.y), (float)(ay * t1.x - by * t1.y));
                    b = make_float2((float)(bx * t0.x + ax * t0.y), (float)(by * t1.x + ay * t1.y));
                }
                x[2 * i] = a;
                x[2 * i + 1] = b;
                if (is_q) {
                    T* dst = q_out + (size_t)t * qo_stride + (size_t)head * hd;
                    store2(dst + 2 * u, a, vec);
                    store2(dst + half + 2 * u, b, vec);
                }
            }
        }
        const bool store = there && !is_q && keep;
        if (__any_sync(0xffffffffu, store)) {
            unsigned char* group = cache + group_at(page, head, off, G, page_size, width);
            unsigned char* codes = group + (is_k ? 0 : 128 * C);
            uint32_t* params = reinterpret_cast<uint32_t*>(group + 256 * C) + 2 * (off & 7) + (is_k ? 0 : 1);
            quantise_store<LANES, UNITS>(x, l, hd, store, codes, off & 7, params);
        }
    }
}

// ---------------------------------------------------------------------------------------------
// Read back: the keys and values that the cache holds at the given slots, m + s n rounded once to the outputs' type.
// A negative slot gives zeros, one behind the pool NaN. One thread per row, kv head and 4 numbers of the key and of the value. Bound: memory.
// ---------------------------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(256)
kv4_read_kernel(const unsigned char* __restrict__ cache, long long num_slots, const int* __restrict__ slots, T* __restrict__ k_out,
                long long k_stride, T* __restrict__ v_out, long long v_stride, long long items, int G, int hd, int page_size) {
    pdl_launch_dependents();
    pdl_wait(31);
    const int quads = hd >> 2, C = chunks(hd);
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < items; i += (long long)gridDim.x * 256) {
        const int u = (int)(i % quads);
        const long long rh = i / quads;
        const int head = (int)(rh % G);
        const long long t = rh / G;
        const int slot = slots[t];
        float kv[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (slot >= num_slots) {
            for (int j = 0; j < 8; ++j) kv[j] = NAN;
        } else if (slot >= 0) {
            const int page = slot / page_size, off = slot - page * page_size;
            const unsigned char* group = cache + group_at(page, head, off, G, page_size, token_bytes(hd));
            const int at = (u >> 3) * 128 + (off & 7) * 16 + (u & 7) * 2;
            const uint2 p = *reinterpret_cast<const uint2*>(group + 256 * C + 8 * (off & 7));
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const unsigned short n = *reinterpret_cast<const unsigned short*>(group + w * 128 * C + at);
                const float2 sm = scale_min(w ? p.y : p.x);
#pragma unroll
                for (int j = 0; j < 4; ++j) kv[4 * w + j] = fmaf((float)(n >> (4 * j) & 15), sm.x, sm.y);
            }
        }
        T* ko = k_out + t * k_stride + (size_t)head * hd + 4 * u;
        T* vo = v_out + t * v_stride + (size_t)head * hd + 4 * u;
#pragma unroll
        for (int j = 0; j < 4; ++j) { st_f(ko + j, kv[j]); st_f(vo + j, kv[4 + j]); }
    }
}

// ---------------------------------------------------------------------------------------------
// Attention in 32-bit arithmetic, any head size up to 256 and any number of heads per kv head: the float32 engine's kernel, and the one
// for portions of head sizes that the tensor-core kernel does not take.
//
// One block: ROWS rows (token, head of the group) of one request and kv head, over KEYS keys at a time: codes become numbers in
// shared memory once per tile, each of 256 threads takes 4 rows x 1 key of the scores and 4 rows x DP / 64 numbers of the sums, the maximum
// and the sum of a row run along in shared memory. `splits` blocks share a request's keys (single tokens); the last one to arrive adds their
// partial results in the order of the keys, so the result does not depend on who that is.
// Bound: the FMA pipe's operands in shared memory.
// ---------------------------------------------------------------------------------------------
constexpr int ROWS = 16, KEYS = 64, FLEX_THREADS = 256;

struct Batch {
    const int* positions;        // single tokens: row s is request s at this position (-1: a padding row). Otherwise null
    const int* seq_starts;
    const int* context_lens;
    const int* block_tables;
    int max_pages, num_pages, page_size, window, H, G, hd;
    float scale;
};

template <int DP> constexpr size_t flex_smem() {
    return sizeof(float) * ((size_t)KEYS * (DP + 4) + (size_t)KEYS * DP + ROWS * DP + KEYS * ROWS + 3 * ROWS);
}

template <typename T, int DP>
__global__ void __launch_bounds__(FLEX_THREADS)
kv4_attend_kernel(const T* __restrict__ q, long long q_stride, T* __restrict__ out, long long out_stride, const unsigned char* __restrict__ cache,
                  Batch b, int splits, float* __restrict__ partials, int* __restrict__ arrived) {
    extern __shared__ float4 smem4[];
    float* sK = reinterpret_cast<float*>(smem4);           // [KEYS][DP + 4]
    float* sV = sK + KEYS * (DP + 4);                      // [KEYS][DP]
    float* sQ = sV + KEYS * DP;                            // [ROWS][DP]
    float* sP = sQ + ROWS * DP;                            // [KEYS][ROWS]
    float* sM = sP + KEYS * ROWS;                          // [ROWS] running maximum
    float* sL = sM + ROWS;                                 // [ROWS] running sum
    float* sA = sL + ROWS;                                 // [ROWS] factor of this tile for what came before
    __shared__ int is_last;
    pdl_launch_dependents();
    pdl_wait(32);
    const int seq = blockIdx.z / splits, split = blockIdx.z % splits, g = blockIdx.y;
    const int group = b.H / b.G, hd = b.hd, tid = threadIdx.x;
    const int row0 = b.positions ? seq : b.seq_starts[seq];
    const int tokens = b.positions ? 1 : b.seq_starts[seq + 1] - row0;
    const int ctx = b.positions ? b.positions[seq] : b.context_lens[seq];
    const int total = tokens * group, tile0 = blockIdx.x * ROWS;
    if (tile0 >= total) return;
    const int nrows = min(ROWS, total - tile0);
    const int last_tok = (tile0 + nrows - 1) / group, first_tok = tile0 / group;
    const int hi = ctx + last_tok + 1;                                                    // keys any row sees: [lo, hi)
    const int lo = b.window ? max(0, ctx + first_tok - b.window + 1) : 0;
    if (hi <= 0) {                                                                        // a padding row sees nothing
        if (split == 0)
            for (int i = tid; i < nrows * hd; i += FLEX_THREADS) {
                const int r = tile0 + i / hd;
                st_f(out + (size_t)(row0 + r / group) * out_stride + (size_t)(g * group + r % group) * hd + i % hd, 0.f);
            }
        return;
    }
    // this block's tiles of keys
    const int t_lo = lo / KEYS, t_hi = (hi + KEYS - 1) / KEYS;
    const int share = (t_hi - t_lo + splits - 1) / splits;
    const int t0 = t_lo + split * share, t1 = min(t_hi, t0 + share);
    const int used = (t_hi - t_lo + share - 1) / share;                                  // splits that have keys
    if (t0 >= t1) return;

    for (int i = tid; i < ROWS * DP; i += FLEX_THREADS) {
        const int r = i / DP, d = i % DP, rr = tile0 + r;
        sQ[i] = (r < nrows && d < hd) ? ld_f(q + (size_t)(row0 + rr / group) * q_stride + (size_t)(g * group + rr % group) * hd + d) * b.scale : 0.f;
    }
    if (tid < ROWS) { sM[tid] = -INFINITY; sL[tid] = 0.f; }
    constexpr int ND = DP / 64;                            // numbers of the sums per thread and row
    float acc[4][ND];
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int d = 0; d < ND; ++d) acc[r][d] = 0.f;
    const int key = tid & 63, rg = (tid >> 6) * 4;
    const int C = chunks(hd), width = token_bytes(hd);
    const int* bt = b.block_tables + (size_t)seq * b.max_pages;

    for (int tile = t0; tile < t1; ++tile) {
        __syncthreads();
        // a warp fetches 8 keys in turn: 4 lanes per key, each C bytes-of-four at a time
        for (int kk = tid >> 2; kk < KEYS; kk += FLEX_THREADS / 4) {
            const int j = tile * KEYS + kk, part = tid & 3;
            float2 ks = make_float2(0.f, 0.f), vs = ks;
            const unsigned char* grp = nullptr;
            if (j < hi && j >= lo) {
                const int pi = j / b.page_size, off = j - pi * b.page_size;
                const int page = pi < b.max_pages ? bt[pi] : -1;
                if (page >= 0 && page < b.num_pages) {
                    grp = cache + group_at(page, g, off, b.G, b.page_size, width) + (off & 7) * 16;
                    attend_scales(*reinterpret_cast<const uint2*>(grp + 256 * C - (off & 7) * 8), ks, vs);
                } else {
                    ks = make_float2(NAN, NAN);             // a page outside the pool: the rows that see it become NaN
                }
            }
            for (int c = 0; c < C; ++c) {
                const uint32_t kn = grp ? *reinterpret_cast<const uint32_t*>(grp + c * 128 + part * 4) : 0u;
                const uint32_t vn = grp ? *reinterpret_cast<const uint32_t*>(grp + (C + c) * 128 + part * 4) : 0u;
                const int d = c * 32 + part * 8;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    sK[kk * (DP + 4) + d + i] = fmaf((float)(kn >> (4 * i) & 15), ks.x, ks.y);
                    sV[kk * DP + d + i] = fmaf((float)(vn >> (4 * i) & 15), vs.x, vs.y);
                }
            }
        }
        __syncthreads();
        float s[4] = {0.f, 0.f, 0.f, 0.f};
        for (int d = 0; d < hd; d += 4) {
            const float4 kx = *reinterpret_cast<const float4*>(sK + key * (DP + 4) + d);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float4 qx = *reinterpret_cast<const float4*>(sQ + (rg + r) * DP + d);
                s[r] = fmaf(kx.w, qx.w, fmaf(kx.z, qx.z, fmaf(kx.y, qx.y, fmaf(kx.x, qx.x, s[r]))));
            }
        }
        const int j = tile * KEYS + key;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int p = ctx + (tile0 + rg + r) / group;
            const bool seen = rg + r < nrows && j <= p && (!b.window || j > p - b.window);
            sP[key * ROWS + rg + r] = seen ? s[r] : -INFINITY;
        }
        __syncthreads();
        // 16 threads per row: the tile's maximum, the probabilities, their sum
        {
            const int r = tid >> 4, i = tid & 15;
            float x[KEYS / 16], mx = -INFINITY;
#pragma unroll
            for (int n = 0; n < KEYS / 16; ++n) {
                x[n] = sP[(i + 16 * n) * ROWS + r];
                mx = fmaxf(mx, x[n]);
            }
            for (int o = 8; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            const float m0 = sM[r], m1 = fmaxf(m0, mx), use = m1 == -INFINITY ? 0.f : m1;
            float sum = 0.f;
#pragma unroll
            for (int n = 0; n < KEYS / 16; ++n) {
                const float p = expf(x[n] - use);
                sP[(i + 16 * n) * ROWS + r] = p;
                sum += p;
            }
            for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (i == 0) {
                const float a = m0 == -INFINITY ? 0.f : expf(m0 - use);
                sA[r] = a;
                sL[r] = sL[r] * a + sum;
                sM[r] = m1;
            }
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float a = sA[rg + r];
#pragma unroll
            for (int d = 0; d < ND; ++d) acc[r][d] *= a;
        }
        for (int kk = 0; kk < KEYS; ++kk) {
            const float4 p = *reinterpret_cast<const float4*>(sP + kk * ROWS + rg);
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                const float x = sV[kk * DP + key + 64 * d];
                acc[0][d] = fmaf(p.x, x, acc[0][d]);
                acc[1][d] = fmaf(p.y, x, acc[1][d]);
                acc[2][d] = fmaf(p.z, x, acc[2][d]);
                acc[3][d] = fmaf(p.w, x, acc[3][d]);
            }
        }
    }
    if (used > 1) {
        // partial of this split: [ROWS][hd] sums, then maxima and sums of the rows
        const size_t unit = (size_t)(seq * b.G + g) * gridDim.x + blockIdx.x;
        const size_t each = (size_t)ROWS * (hd + 2);
        float* mine = partials + (unit * splits + split) * each;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int d = 0; d < ND; ++d)
                if (key + 64 * d < hd) mine[(rg + r) * hd + key + 64 * d] = acc[r][d];
        if (tid < ROWS) { mine[ROWS * hd + tid] = sM[tid]; mine[ROWS * hd + ROWS + tid] = sL[tid]; }
        __threadfence();
        __syncthreads();
        if (tid == 0) {
            is_last = atomicAdd(arrived + unit, 1) == used - 1;
            if (is_last) arrived[unit] = 0;                // as it was found, for the next launch
        }
        __syncthreads();
        if (!is_last) return;
        __threadfence();
        const float* all = partials + unit * splits * each;
        if (tid < ROWS) {
            float m = -INFINITY;
            for (int s = 0; s < used; ++s) m = fmaxf(m, __ldcg(all + s * each + ROWS * hd + tid));
            sM[tid] = m;
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            float l = 0.f;
#pragma unroll
            for (int d = 0; d < ND; ++d) acc[r][d] = 0.f;
            const float m = sM[rg + r];
            for (int s = 0; s < used; ++s) {
                const float* part = all + s * each;
                const float ms = __ldcg(part + ROWS * hd + rg + r);
                const float a = ms == -INFINITY ? 0.f : expf(ms - m);
                l += a * __ldcg(part + ROWS * hd + ROWS + rg + r);
#pragma unroll
                for (int d = 0; d < ND; ++d)
                    if (key + 64 * d < hd) acc[r][d] = fmaf(a, __ldcg(part + (rg + r) * hd + key + 64 * d), acc[r][d]);
            }
            if (key == 0) sL[rg + r] = l;
        }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 4; ++r)
        if (rg + r < nrows) {
            const int rr = tile0 + rg + r;
            const float l = sL[rg + r], inv = l == 0.f ? 0.f : 1.f / l;
            T* dst = out + (size_t)(row0 + rr / group) * out_stride + (size_t)(g * group + rr % group) * hd;
#pragma unroll
            for (int d = 0; d < ND; ++d)
                if (key + 64 * d < hd) st_f(dst + key + 64 * d, acc[r][d] * inv);
        }
}

template <typename T, int DP>
int launch_attend(const void* q, long long q_stride, void* out, long long out_stride, const unsigned char* cache, const Batch& b, int S,
                  int max_new, int splits, float* partials, int* arrived, cudaStream_t stream) {
    // once per device that the process uses: the attribute belongs to the current one
    static size_t done[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    if (dev >= 64 || !done[dev]) {
        e = cudaFuncSetAttribute(kv4_attend_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)flex_smem<DP>());
        if (e != cudaSuccess) return (int)e;
        if (dev < 64) done[dev] = 1;
    }
    const long long tiles = ((long long)max_new * (b.H / b.G) + ROWS - 1) / ROWS;
    if (tiles > 0x7fffffffLL || b.G > 65535 || (long long)S * splits > 65535) return VOB_ERR_UNSUPPORTED;
    return vob_launch(kv4_attend_kernel<T, DP>, dim3((unsigned)tiles, b.G, S * splits), dim3(FLEX_THREADS), flex_smem<DP>(), stream,
                      (const T*)q, q_stride, (T*)out, out_stride, cache, b, splits, partials, arrived);
}

bool sizes_ok(int H, int G, int hd, int page_size) {
    return H > 0 && G > 0 && H % G == 0 && hd > 0 && hd % 16 == 0 && hd <= 256 && page_size > 0 && page_size % 8 == 0;
}

}  // namespace

// q, q_out [T, H * hd], k, v [T, G * hd] (row strides in elements; q_out may be q). slots int32 [T], or null: nothing is kept.
VOB_EXPORT int vob_kv4_append(const void* q, long long q_stride, void* q_out, long long qo_stride, const void* k, long long k_stride,
                              const void* v, long long v_stride, const int* positions, const int* slots, const float* inv_freq,
                              void* cache, long long num_pages, int code, int T, int H, int G, int hd, int page_size, cudaStream_t stream) {
    if (T <= 0) return 0;
    if (!sizes_ok(H, G, hd, page_size) || num_pages <= 0) return VOB_ERR_BAD_ARG;
    const int es = code == VOB_F32 ? 4 : 2;
    const bool vec = (((uintptr_t)q | (uintptr_t)q_out | (uintptr_t)k | (uintptr_t)v) % (2 * es)) == 0 &&
                     ((q_stride | qo_stride | k_stride | v_stride) % 2) == 0;
    const long long num_slots = num_pages * page_size;
    const int vectors = H + 2 * G, lanes = hd <= 64 ? 16 : 32;
    const int per_pass = (APPEND_THREADS / 32) * (32 / lanes);
    // few tokens: a block per pass over the vectors, so that a decode step's tokens spread over the GPU
    int y = (vectors + per_pass - 1) / per_pass;
    if ((long long)T * y > 4 * 148) y = (int)max(1LL, (long long)(4 * 148) / T);
    const dim3 grid(T, y), block(APPEND_THREADS);
#define VOB_APPEND(L, U)                                                                                                              \
    VOB_DISPATCH_ELEM(code, return vob_launch(kv4_append_kernel<ElemT, L, U>, grid, block, 0, stream, (const ElemT*)q, q_stride,          \
                                              (ElemT*)q_out, qo_stride, (const ElemT*)k, k_stride, (const ElemT*)v, v_stride, positions,  \
                                              slots, inv_freq, (unsigned char*)cache, num_slots, H, G, hd, page_size, vec))
    if (hd <= 64) VOB_APPEND(16, 1);
    if (hd <= 128) VOB_APPEND(32, 1);
    VOB_APPEND(32, 2);
#undef VOB_APPEND
    return 0;
}

VOB_EXPORT int vob_kv4_read(const void* cache, long long num_pages, const int* slots, void* k_out, long long k_stride, void* v_out,
                            long long v_stride, int code, int T, int G, int hd, int page_size, cudaStream_t stream) {
    if (T <= 0) return 0;
    if (!sizes_ok(G, G, hd, page_size) || num_pages <= 0) return VOB_ERR_BAD_ARG;
    const long long items = (long long)T * G * (hd >> 2);
    const long long blocks = (items + 255) / 256;
    VOB_DISPATCH_ELEM(code, return vob_launch(kv4_read_kernel<ElemT>, dim3((unsigned)min(blocks, 148LL * 16)), dim3(256), 0, stream,
                                              (const unsigned char*)cache, num_pages * page_size, slots, (ElemT*)k_out, k_stride,
                                              (ElemT*)v_out, v_stride, items, G, hd, page_size));
    return 0;
}

// Attention in 32-bit arithmetic. Single tokens: `positions` int32 [S] (row s of q is request s); otherwise seq_starts int32 [S + 1] and
// context_lens int32 [S]. `partials` (splits > 1): S * G * row tiles * splits * 16 * (hd + 2) floats; `arrived`: S * G * row tiles zeros.
VOB_EXPORT int vob_kv4_attend(const void* q, long long q_stride, void* out, long long out_stride, const void* cache, long long num_pages,
                              const int* block_tables, int max_pages, const int* positions, const int* seq_starts, const int* context_lens,
                              int S, int max_new, int H, int G, int hd, int page_size, float scale, int window, int code, int splits,
                              float* partials, int* arrived, cudaStream_t stream) {
    if (S <= 0 || max_new <= 0) return 0;
    if (!sizes_ok(H, G, hd, page_size) || num_pages <= 0 || num_pages > 0x7fffffffLL || splits <= 0 || window < 0) return VOB_ERR_BAD_ARG;
    if (splits > 1 && (!partials || !arrived || !positions)) return VOB_ERR_BAD_ARG;
    if (!positions && (!seq_starts || !context_lens)) return VOB_ERR_BAD_ARG;
    Batch b = {positions, seq_starts, context_lens, block_tables, max_pages, (int)num_pages, page_size, window, H, G, hd, scale};
    const unsigned char* c = (const unsigned char*)cache;
#define VOB_ATTEND(DP) VOB_DISPATCH_ELEM(code, return launch_attend<ElemT, DP>(q, q_stride, out, out_stride, c, b, S, max_new, splits, partials, arrived, stream))
    if (hd <= 64) VOB_ATTEND(64);
    if (hd <= 128) VOB_ATTEND(128);
    VOB_ATTEND(256);
#undef VOB_ATTEND
    return 0;
}
