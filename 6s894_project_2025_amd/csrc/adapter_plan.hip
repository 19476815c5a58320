// Tokens of a batch grouped by adapter (mi_adapter_plan): a stable counting sort of the ids and the
// tables of work that the low-rank adapter kernels read (adapter_plan.hpp).
//
// A wavefront takes a contiguous stretch of the tokens, 64 at a time.  Lanes with the same id find each other by
// one ballot per bit of the id (none where all 64 ids are the same, as inside a long request), so a token's
// place among its wavefront's tokens of the same adapter is a count of earlier lanes.  First pass: counts per
// wavefront and adapter in LDS.  A scan over adapters and wavefronts turns them into positions.  Second pass:
// the tokens to their positions.  So the order is stable, and the same whatever the timing.
// Up to 4096 tokens one workgroup of 16 wavefronts does everything in one launch; beyond, workgroups of four
// wavefronts leave their counts in memory and a second launch reads them all (32768 tokens of 32 adapters: 52 us
// with one workgroup, 10 with two launches).
// Bound: latency.  The bytes (8 a token) would take 0.05 us; what is left are two dependent passes over a stretch,
// with a scan and its barriers between them, and the launches (256 tokens of 64 adapters: 7 us).
#include "adapter_plan.hpp"

namespace mi {
namespace adapters {
namespace {

constexpr uint32_t kAhead = 4;  // groups of 64 ids requested together

typedef uint32_t Four __attribute__((ext_vector_type(4)));

// Inclusive scan of four values per thread over the workgroup.
__device__ __forceinline__ Four block_scan(Four v, Four* wave_sums)
{
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    for (uint32_t d = 1; d < 64u; d <<= 1) {
        Four up;
#pragma unroll
        for (int i = 0; i < 4; ++i) up[i] = __shfl_up(v[i], d);
        if (lane >= d) v += up;
    }
    __syncthreads();  // the sums of an earlier scan may still be read
    if (lane == 63u) wave_sums[wave] = v;
    __syncthreads();
    for (uint32_t w = 0; w < wave; ++w) v += wave_sums[w];
    return v;
}

// Calls f(token, key, lanes with the same key) for the live lanes of each 64 of the tokens [t0, t1), in order.
template <class Id, class F>
__device__ __forceinline__ void for_groups(const Id* ids, uint32_t t0, uint32_t t1, uint32_t n, uint32_t key_bits, F f)
{
    const uint32_t lane = threadIdx.x & 63u;
    for (uint32_t base = t0; base < t1; base += 64u * kAhead) {
        Id id[kAhead];
#pragma unroll
        for (uint32_t k = 0; k < kAhead; ++k) {
            const uint32_t t = base + 64u * k + lane;
            id[k] = ids[t < t1 ? t : t0];
        }
#pragma unroll
        for (uint32_t k = 0; k < kAhead; ++k) {
            const uint32_t t = base + 64u * k + lane;
            const bool live = t < t1;
            const uint32_t key = id[k] >= 0 && id[k] < (Id)n ? (uint32_t)id[k] : n;
            uint64_t same = __ballot(live);
            if (__ballot(live && key != (uint32_t)__builtin_amdgcn_readfirstlane(key)))  // the first lane is live, or none is
                for (uint32_t b = 0; b < key_bits; ++b) {
                    const uint64_t ones = __ballot(key >> b & 1u);
                    same &= key >> b & 1u ? ones : ~ones;
                }
            if (live) f(t, key, same);
            __builtin_amdgcn_wave_barrier();
        }
    }
}

// Counts of the wavefront's tokens by key.
template <class Id>
__device__ __forceinline__ void count_keys(const Id* ids, uint32_t t0, uint32_t t1, uint32_t n, uint32_t key_bits, uint32_t* hist)
{
    const uint32_t lane = threadIdx.x & 63u;
    for_groups(ids, t0, t1, n, key_bits, [&](uint32_t, uint32_t key, uint64_t same) {
        if ((same >> lane) == 1ull) hist[key] += (uint32_t)__popcll(same);  // the last lane of its key
    });
}

// The wavefront's tokens to their places; at[key]: the place of its next token of that key.
template <class Id>
__device__ __forceinline__ void place_tokens(const Id* ids, uint32_t t0, uint32_t t1, uint32_t n, uint32_t key_bits, uint32_t* at, int32_t* order)
{
    const uint32_t lane = threadIdx.x & 63u;
    for_groups(ids, t0, t1, n, key_bits, [&](uint32_t t, uint32_t key, uint64_t same) {
        const uint32_t place = at[key] + (uint32_t)__popcll(same & ((1ull << lane) - 1ull));
        order[place] = (int32_t)t;
        __builtin_amdgcn_wave_barrier();
        if ((same >> lane) == 1ull) at[key] = place + 1u;  // once all its lanes have read
    });
}

// The scans over the adapters: from the counts of each, in LDS, to the first position, tile, chunk and slot.
struct Scans {
    Four* wave_sums;                           // [wavefronts]
    uint32_t *start, *tile, *chunk, *slot;     // [keys + 1] each
    __device__ __forceinline__ Scans(uint32_t* lds, uint32_t waves, uint32_t keys)
        : wave_sums(reinterpret_cast<Four*>(lds)), start(lds + 4u * waves), tile(start + keys + 1u), chunk(tile + keys + 1u), slot(chunk + keys + 1u)
    {
    }
    template <class Total>  // total(key): called once for each key, by one thread
    __device__ __forceinline__ void run(const PlanLayout& L, uint32_t keys, Total total)
    {
        uint32_t* const out[4] = {start, tile, chunk, slot};
        Four carry = {0u, 0u, 0u, 0u};
        for (uint32_t base = 0; base < keys; base += blockDim.x) {
            const uint32_t k = base + threadIdx.x;
            const uint32_t count = k < keys ? total(k) : 0u;
            const uint32_t chunks = k + 1u < keys ? (count + L.chunk - 1u) / L.chunk : 0u;  // not for tokens without an adapter
            const Four end = carry + block_scan(Four{count, (count + kTile - 1u) / kTile, chunks, chunks > 1u ? chunks : 0u}, wave_sums);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (k < keys) out[i][k + 1u] = end[i];
                if (k == 0u) out[i][0] = 0u;
            }
            __syncthreads();
            const uint32_t last = base + blockDim.x < keys ? base + blockDim.x : keys;
            carry = Four{start[last], tile[last], chunk[last], slot[last]};
        }
    }
    __device__ __forceinline__ void write_tables(const PlanLayout& L, uint32_t keys, int32_t* plan) const
    {
        for (uint32_t k = threadIdx.x; k < keys; k += blockDim.x) {
            plan[L.starts + k] = (int32_t)start[k];
            if (k + 1u < keys) plan[L.slot_start + k] = (int32_t)slot[k];
        }
        if (threadIdx.x == 0) {
            plan[L.counts] = (int32_t)tile[keys];
            plan[L.counts + 1u] = (int32_t)chunk[keys];
        }
        // entry i belongs to the adapter whose range of entries holds i
        auto owner = [&](const uint32_t* s, uint32_t i) {
            uint32_t lo = 0, hi = keys;  // s[lo] <= i < s[hi]
            while (hi - lo > 1u) {
                const uint32_t mid = (lo + hi) / 2u;
                if (s[mid] <= i) lo = mid; else hi = mid;
            }
            return lo;
        };
        Tile* tiles = reinterpret_cast<Tile*>(plan);
        for (uint32_t i = threadIdx.x; i < tile[keys]; i += blockDim.x) {
            const uint32_t k = owner(tile, i), first = start[k] + (i - tile[k]) * kTile, left = start[k + 1u] - first;
            tiles[i] = Tile{(int32_t)k, (int32_t)first, (int32_t)(left < kTile ? left : kTile), 0};
        }
        Chunk* chunks = reinterpret_cast<Chunk*>(plan + L.chunks);
        for (uint32_t i = threadIdx.x; i < chunk[keys]; i += blockDim.x) {
            const uint32_t k = owner(chunk, i), c = i - chunk[k], first = start[k] + c * L.chunk, left = start[k + 1u] - first;
            const bool many = slot[k + 1u] > slot[k];
            chunks[i] = Chunk{(int32_t)k, (int32_t)first, (int32_t)(left < L.chunk ? left : L.chunk), many ? (int32_t)(slot[k] + c) : -1,
                              (int32_t)(tile[k] + c * (L.chunk / kTile)), {0, 0, 0}};
        }
    }
};

// LDS of a kernel with `waves` wavefronts.
constexpr uint32_t lds_bytes(uint32_t waves, uint32_t keys) { return (4u * waves + 4u * (keys + 1u) + waves * keys) * 4u; }

// A wavefront's share [t0, t1) of the tokens [from, to).
template <uint32_t WAVES>
__device__ __forceinline__ void share(uint32_t from, uint32_t to, uint32_t& t0, uint32_t& t1)
{
    const uint32_t per = ((to - from + WAVES - 1u) / WAVES + 63u) / 64u * 64u, begin = from + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * per;
    t0 = begin < to ? begin : to;
    t1 = to - t0 < per ? to : t0 + per;
}

template <class Id>
__global__ void __launch_bounds__(1024) adapter_plan_kernel(const Id* ids, uint32_t T, uint32_t n, uint32_t key_bits, int32_t* plan)
{
    constexpr uint32_t WAVES = 16;
    extern __shared__ __attribute__((aligned(16))) uint32_t lds[];
    const PlanLayout L(T, n);
    const uint32_t keys = n + 1u;
    Scans scans(lds, WAVES, keys);
    uint32_t* const hist = scans.slot + keys + 1u;  // [WAVES][keys]
    uint32_t* const mine = hist + (threadIdx.x >> 6) * keys;
    for (uint32_t i = threadIdx.x; i < WAVES * keys; i += blockDim.x) hist[i] = 0u;
    __syncthreads();
    uint32_t t0, t1;
    share<WAVES>(0, T, t0, t1);
    count_keys(ids, t0, t1, n, key_bits, mine);
    __syncthreads();
    scans.run(L, keys, [&](uint32_t k) {
        uint32_t total = 0;
        for (uint32_t w = 0; w < WAVES; ++w) {
            const uint32_t c = hist[w * keys + k];
            hist[w * keys + k] = total;
            total += c;
        }
        return total;
    });
    for (uint32_t i = threadIdx.x; i < WAVES * keys; i += blockDim.x) hist[i] += scans.start[i % keys];
    __syncthreads();
    place_tokens(ids, t0, t1, n, key_bits, mine, plan + L.order);
    scans.write_tables(L, keys, plan);
}

// The tokens of workgroup g of L.groups.
__device__ __forceinline__ void group_range(const PlanLayout& L, uint32_t T, uint32_t g, uint32_t& from, uint32_t& to)
{
    const uint32_t per = ((T + L.groups - 1u) / L.groups + 63u) / 64u * 64u;
    from = g * per < T ? g * per : T;
    to = T - from < per ? T : from + per;
}

template <class Id>
__global__ void __launch_bounds__(256) count_kernel(const Id* ids, uint32_t T, uint32_t n, uint32_t key_bits, int32_t* plan)
{
    constexpr uint32_t WAVES = 4;
    extern __shared__ __attribute__((aligned(16))) uint32_t lds[];
    const PlanLayout L(T, n);
    const uint32_t keys = n + 1u;
    for (uint32_t i = threadIdx.x; i < WAVES * keys; i += blockDim.x) lds[i] = 0u;
    __syncthreads();
    uint32_t from, to, t0, t1;
    group_range(L, T, blockIdx.x, from, to);
    share<WAVES>(from, to, t0, t1);
    count_keys(ids, t0, t1, n, key_bits, lds + (threadIdx.x >> 6) * keys);
    __syncthreads();
    for (uint32_t k = threadIdx.x; k < keys; k += blockDim.x)
        plan[L.histograms + (uint64_t)blockIdx.x * keys + k] = (int32_t)(lds[k] + lds[keys + k] + lds[2u * keys + k] + lds[3u * keys + k]);
}

// Workgroups 0 ... groups - 1 place their tokens, one more writes the tables.
template <class Id>
__global__ void __launch_bounds__(256) place_kernel(const Id* ids, uint32_t T, uint32_t n, uint32_t key_bits, int32_t* plan)
{
    constexpr uint32_t WAVES = 4;
    extern __shared__ __attribute__((aligned(16))) uint32_t lds[];
    const PlanLayout L(T, n);
    const uint32_t keys = n + 1u;
    Scans scans(lds, WAVES, keys);
    uint32_t* const hist = scans.slot + keys + 1u;  // [WAVES][keys]
    uint32_t* const mine = hist + (threadIdx.x >> 6) * keys;
    for (uint32_t i = threadIdx.x; i < WAVES * keys; i += blockDim.x) hist[i] = 0u;
    __syncthreads();
    uint32_t from, to, t0, t1;
    group_range(L, T, blockIdx.x < L.groups ? blockIdx.x : 0u, from, to);
    share<WAVES>(from, to, t0, t1);
    if (blockIdx.x < L.groups) count_keys(ids, t0, t1, n, key_bits, mine);
    __syncthreads();
    const int32_t* all = plan + L.histograms;
    scans.run(L, keys, [&](uint32_t k) {
        uint32_t before = 0, total = 0;
#pragma unroll 8
        for (uint32_t g = 0; g < L.groups; ++g) {
            const uint32_t c = (uint32_t)all[(uint64_t)g * keys + k];
            total += c;
            before += g < blockIdx.x ? c : 0u;
        }
        for (uint32_t w = 0; w < WAVES; ++w) {
            const uint32_t c = hist[w * keys + k];
            hist[w * keys + k] = before;
            before += c;
        }
        return total;
    });
    if (blockIdx.x == L.groups) {
        scans.write_tables(L, keys, plan);
        return;
    }
    for (uint32_t i = threadIdx.x; i < WAVES * keys; i += blockDim.x) hist[i] += scans.start[i % keys];
    __syncthreads();
    place_tokens(ids, t0, t1, n, key_bits, mine, plan + L.order);
}

template <class Id>
int make_plan(const Id* ids, uint32_t T, uint32_t n, int32_t* plan, hipStream_t s)
{
    const PlanLayout L(T, n);
    uint32_t key_bits = 0;
    while (n >> key_bits) ++key_bits;
    if (L.groups == 0) {
        const uint32_t bytes = lds_bytes(16, n + 1u);
        if (bytes > 65536u && hipFuncSetAttribute(reinterpret_cast<const void*>(adapter_plan_kernel<Id>), hipFuncAttributeMaxDynamicSharedMemorySize,
                                                  (int)bytes) != hipSuccess)
            return MI_ERR_LAUNCH;
        hipLaunchKernelGGL((adapter_plan_kernel<Id>), dim3(1), dim3(1024), bytes, s, ids, T, n, key_bits, plan);
        return launch_status();
    }
    hipLaunchKernelGGL((count_kernel<Id>), dim3(L.groups), dim3(256), lds_bytes(4, n + 1u), s, ids, T, n, key_bits, plan);
    const int st = launch_status();
    if (st != MI_OK) return st;
    hipLaunchKernelGGL((place_kernel<Id>), dim3(L.groups + 1u), dim3(256), lds_bytes(4, n + 1u), s, ids, T, n, key_bits, plan);
    return launch_status();
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
    hipStream_t s = static_cast<hipStream_t>(stream);
    return id_bits == 32 ? make_plan(static_cast<const int32_t*>(ids), (uint32_t)tokens, n_adapters, plan, s)
                         : make_plan(static_cast<const int64_t*>(ids), (uint32_t)tokens, n_adapters, plan, s);
}
