// Tokens of a batch grouped by adapter (mi_adapter_plan): a stable counting sort of the ids and the
// tables of work that the low-rank adapter kernels read (adapter_plan.hpp).
//
// One workgroup of 16 wavefronts; each takes one contiguous stretch of the tokens.  First pass: counts
// per (wavefront, adapter) in LDS.  A scan over adapters and wavefronts turns them into the position of
// each wavefront's first token of each adapter.  Second pass: 64 tokens at a time, a token's place among
// the wavefront's tokens of its adapter is the number of earlier lanes with the same id, found by one
// ballot per bit of the id.  So the order is stable, and the same whatever the timing.
#include "adapter_plan.hpp"

namespace mi {
namespace adapters {
namespace {

constexpr uint32_t kThreads = 1024, kWaves = kThreads / 64u;

// Inclusive scan of one value per thread over the workgroup.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* wave_sums)
{
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    for (uint32_t d = 1; d < 64u; d <<= 1) {
        const uint32_t up = __shfl_up(v, d);
        if (lane >= d) v += up;
    }
    __syncthreads();  // the sums of an earlier scan may still be read
    if (lane == 63u) wave_sums[wave] = v;
    __syncthreads();
    for (uint32_t w = 0; w < wave; ++w) v += wave_sums[w];
    return v;
}

template <class Id>
__device__ __forceinline__ uint32_t key_of(const Id* ids, uint64_t t, uint32_t n)
{
    const Id id = ids[t];
    return id >= 0 && id < (Id)n ? (uint32_t)id : n;
}

template <class Id>
__global__ void __launch_bounds__(1024) adapter_plan_kernel(const Id* ids, uint32_t T, uint32_t n, uint32_t key_bits, int32_t* plan)
{
    extern __shared__ uint32_t lds[];
    const PlanLayout L(T, n);
    const uint32_t keys = n + 1u;
    uint32_t* hist = lds;                       // [kWaves][keys]
    uint32_t* start = hist + kWaves * keys;     // [keys + 1]: first position of an adapter
    uint32_t* tile_start = start + keys + 1u;   // [keys + 1]
    uint32_t* chunk_start = tile_start + keys + 1u;
    uint32_t* slot_start = chunk_start + keys + 1u;
    uint32_t* wave_sums = slot_start + keys + 1u;
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;

    for (uint32_t i = threadIdx.x; i < kWaves * keys; i += kThreads) hist[i] = 0u;
    __syncthreads();
    const uint32_t per_wave = (((T + kWaves - 1u) / kWaves) + 63u) / 64u * 64u;
    const uint32_t t0 = wave * per_wave < T ? wave * per_wave : T;
    const uint32_t t1 = t0 + per_wave < T ? t0 + per_wave : T;
    for (uint32_t t = t0 + lane; t < t1; t += 64u) atomicAdd(&hist[wave * keys + key_of(ids, t, n)], 1u);
    __syncthreads();

    // scans over the adapters, kThreads of them at a time
    uint32_t carry[4] = {0u, 0u, 0u, 0u};
    for (uint32_t base = 0; base < keys; base += kThreads) {
        const uint32_t k = base + threadIdx.x;
        uint32_t total = 0;
        if (k < keys)
            for (uint32_t w = 0; w < kWaves; ++w) {
                const uint32_t c = hist[w * keys + k];
                hist[w * keys + k] = total;
                total += c;
            }
        const uint32_t chunks = k < n ? (total + L.chunk - 1u) / L.chunk : 0u;
        const uint32_t add[4] = {total, (total + kTile - 1u) / kTile, chunks, chunks > 1u ? chunks : 0u};
        uint32_t* out[4] = {start, tile_start, chunk_start, slot_start};
        for (int i = 0; i < 4; ++i) {
            const uint32_t end = carry[i] + block_scan(add[i], wave_sums);
            if (k < keys) out[i][k + 1u] = end;
            __syncthreads();
            carry[i] = out[i][base + kThreads < keys ? base + kThreads : keys];
        }
        if (k == 0u)
            for (int i = 0; i < 4; ++i) out[i][0] = 0u;
    }
    __syncthreads();

    // the grouped order
    for (uint32_t t = t0; t < t1; t += 64u) {
        const bool live = t + lane < t1;
        const uint32_t key = live ? key_of(ids, t + lane, n) : 0u;
        uint64_t same = __ballot(live);
        for (uint32_t b = 0; b < key_bits; ++b) {
            const uint64_t ones = __ballot(key >> b & 1u);
            same &= key >> b & 1u ? ones : ~ones;
        }
        if (live) {
            const uint32_t before = (uint32_t)__popcll(same & ((1ull << lane) - 1ull));
            uint32_t* at = &hist[wave * keys + key];
            const uint32_t place = *at + before;
            plan[L.order + start[key] + place] = (int32_t)(t + lane);
            __builtin_amdgcn_wave_barrier();
            if ((same >> lane) == 1ull) *at = place + 1u;  // last lane of its adapter, once all have read
        }
        __builtin_amdgcn_wave_barrier();
    }

    for (uint32_t k = threadIdx.x; k < keys; k += kThreads) {
        plan[L.starts + k] = (int32_t)start[k];
        if (k < n) plan[L.slot_start + k] = (int32_t)slot_start[k];
    }
    if (threadIdx.x == 0) {
        plan[L.counts] = (int32_t)tile_start[keys];
        plan[L.counts + 1u] = (int32_t)chunk_start[keys];
    }
    // tables: entry i belongs to the adapter whose range of entries holds i
    auto owner = [&](const uint32_t* s, uint32_t i) {
        uint32_t lo = 0, hi = keys;  // s[lo] <= i < s[hi]
        while (hi - lo > 1u) {
            const uint32_t mid = (lo + hi) / 2u;
            if (s[mid] <= i) lo = mid; else hi = mid;
        }
        return lo;
    };
    Tile* tiles = reinterpret_cast<Tile*>(plan);
    for (uint32_t i = threadIdx.x; i < tile_start[keys]; i += kThreads) {
        const uint32_t k = owner(tile_start, i), first = start[k] + (i - tile_start[k]) * kTile;
        const uint32_t left = start[k + 1u] - first;
        tiles[i] = Tile{(int32_t)k, (int32_t)first, (int32_t)(left < kTile ? left : kTile), 0};
    }
    Chunk* chunks = reinterpret_cast<Chunk*>(plan + L.chunks);
    for (uint32_t i = threadIdx.x; i < chunk_start[keys]; i += kThreads) {
        const uint32_t k = owner(chunk_start, i), c = i - chunk_start[k], first = start[k] + c * L.chunk;
        const uint32_t left = start[k + 1u] - first;
        const bool many = slot_start[k + 1u] > slot_start[k];
        chunks[i] = Chunk{(int32_t)k, (int32_t)first, (int32_t)(left < L.chunk ? left : L.chunk),
                          many ? (int32_t)(slot_start[k] + c) : -1, (int32_t)(tile_start[k] + c * (L.chunk / kTile)), {0, 0, 0}};
    }
}

}  // namespace
}  // namespace adapters
}  // namespace mi

extern "C" int mi_adapter_plan_layout(uint64_t tokens, uint32_t n_adapters, uint64_t* layout)
{
    using namespace mi;
    if (!layout) return MI_ERR_NULL;
    if (tokens > adapters::kMaxTokens || n_adapters < 1u || n_adapters > adapters::kMaxAdapters) return MI_ERR_SHAPE;
    const adapters::PlanLayout L(tokens, n_adapters);
    layout[0] = L.size;
    layout[1] = L.order;
    layout[2] = L.starts;
    return MI_OK;
}

extern "C" int mi_adapter_plan(const void* ids, int id_bits, uint64_t tokens, uint32_t n_adapters, int32_t* plan, void* stream)
{
    using namespace mi;
    using namespace mi::adapters;
    if (id_bits != 32 && id_bits != 64) return MI_ERR_DTYPE;
    if (tokens > kMaxTokens || n_adapters < 1u || n_adapters > kMaxAdapters) return MI_ERR_SHAPE;
    if (!plan || (tokens && !ids)) return MI_ERR_NULL;
    if (!aligned16(plan) || reinterpret_cast<uintptr_t>(ids) % (id_bits / 8)) return MI_ERR_ALIGN;
    const uint32_t keys = n_adapters + 1u;
    const uint32_t bytes = (kWaves * keys + 4u * (keys + 1u) + kWaves) * 4u;
    uint32_t key_bits = 0;
    while (n_adapters >> key_bits) ++key_bits;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (bytes > 65536u) {
        const void* kern = id_bits == 32 ? reinterpret_cast<const void*>(adapter_plan_kernel<int32_t>)
                                         : reinterpret_cast<const void*>(adapter_plan_kernel<int64_t>);
        if (hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) != hipSuccess) return MI_ERR_LAUNCH;
    }
    if (id_bits == 32)
        hipLaunchKernelGGL((adapter_plan_kernel<int32_t>), dim3(1), dim3(kThreads), bytes, s, static_cast<const int32_t*>(ids),
                           (uint32_t)tokens, n_adapters, key_bits, plan);
    else
        hipLaunchKernelGGL((adapter_plan_kernel<int64_t>), dim3(1), dim3(kThreads), bytes, s, static_cast<const int64_t*>(ids),
                           (uint32_t)tokens, n_adapters, key_bits, plan);
    return launch_status();
}
