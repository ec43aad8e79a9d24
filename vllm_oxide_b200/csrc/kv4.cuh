// The cache that holds keys and values in 4 bits: its layout and its numbers, shared by the kernels that write and read it.
//
// Of a token's key (value) of one kv head, D numbers x, are kept a scale s = bf16(max x / 15 - min x / 15), a minimum
// m = bf16(min x) and a code n = round((x - m) / s) in 0 .. 15 per number; a code stands for m + s n. One scale and one minimum per
// vector: 8 bytes for a key and its value beside D bytes of codes (136 bytes at D = 128, where 16 bits take 512), and the scores and sums
// can be taken on the codes alone, s and m coming in once per (row, key).
//
// A layer's cache is uint8 [pages, kv heads, page size, W], W = 32 C + 8 bytes per token, C = ceil(D / 32) chunks of 32 numbers.
// Eight tokens of one page and kv head, positions 8i .. 8i + 7, lie together (page sizes are multiples of 8), so that any run of them is
// contiguous whatever the page size, and a chunk of eight tokens is 128 bytes that ldmatrix reads without a bank conflict:
//   [C][8 tokens][16 bytes]   codes of the keys; byte b of a chunk: number 2b in its low four bits, 2b + 1 in its high ones
//   [C][8 tokens][16 bytes]   codes of the values
//   [8 tokens][4 bfloat16]    s and m of the key, s and m of the value
// What D leaves of the last chunk holds zeros.
#pragma once
#include "common.cuh"

namespace vob_kv4 {

constexpr int GROUP = 8;                                                            // tokens that lie together
__host__ __device__ constexpr int chunks(int hd) { return (hd + 31) / 32; }
__host__ __device__ constexpr int token_bytes(int hd) { return 32 * chunks(hd) + 8; }

// First byte of the group of eight tokens that holds token `off` of a page.
__device__ __forceinline__ size_t group_at(size_t page, int head, int off, int kv_heads, int page_size, int width) {
    return ((page * kv_heads + head) * page_size + (off & ~7)) * (size_t)width;
}

// s and m of a key or value from the two bfloat16 of one 32-bit word.
__device__ __forceinline__ float2 scale_min(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ bool is_finite2(float2 a) { return isfinite(a.x) && isfinite(a.y); }

// s and m of a key and its value, as attention takes them. A value that is not finite (its token's projection was not) is taken as 0
// and its key as NaN: the rows that see the token become NaN through their scores, and no other row does, as 0 * NaN would make them
// where a product is taken over tokens that a row's mask hides.
__device__ __forceinline__ void attend_scales(uint2 p, float2& key, float2& val) {
    key = scale_min(p.x);
    val = scale_min(p.y);
    if (!is_finite2(val)) {
        key = make_float2(NAN, NAN);
        val = make_float2(0.f, 0.f);
    }
}

// ---------------------------------------------------------------------------------------------
// Blocks that share the keys of a row form a cluster, each with its part of the sums in its own shared memory; at the end every block joins
// a share of the rows, reading the others'.
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_blocks() { uint32_t n; asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(n)); return n; }
__device__ __forceinline__ uint32_t cluster_rank() { uint32_t n; asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(n)); return n; }
// All threads of all its blocks; what they wrote before is seen behind it. No wait here depends on anything but the blocks' own bounded loops.
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// A float of block `rank`'s shared memory, where this block has `p`.
__device__ __forceinline__ float ld_cluster(const float* p, uint32_t rank) {
    uint32_t at;
    float x;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(at) : "memory");
    return x;
}
__device__ __forceinline__ float4 ld_cluster4(const float* p, uint32_t rank) {
    uint32_t at;
    float4 x;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "r"(at) : "memory");
    return x;
}
// The weight of a part of a row's keys whose maximum (base 2) is `mine`: a part without keys has nothing to weigh (its sums are 0); one whose keys all
// gave NaN has no maximum either, and stays NaN.
__device__ __forceinline__ float part_weight(float mine, float all) { return mine == -INFINITY ? 1.f : exp2f(mine - all); }

// Blocks that share a row's keys, up to the 8 of a portable cluster and to `most`, so that there are `wanted` in all.
static inline int key_parts(long long blocks, long long wanted, long long most) {
    int n = 1;
    while (n < 8 && blocks * n < wanted && 2 * n <= most) n *= 2;
    return n;
}
// Clusters of `parts` blocks that the current device runs at once.
template <typename... P>
static inline cudaError_t cluster_room(void (*kernel)(P...), int parts, dim3 block, size_t smem, int* clusters) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(parts * 148);
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = parts;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaOccupancyMaxActiveClusters(clusters, kernel, &cfg);
}
template <typename... P, typename... A>
static inline int launch_clusters(void (*kernel)(P...), dim3 grid, int parts, dim3 block, size_t smem, cudaStream_t stream, A&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = parts;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = g_vob_pdl ? 2 : 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
    return e != cudaSuccess ? (int)e : vob_launch_status();
}

}  // namespace vob_kv4
