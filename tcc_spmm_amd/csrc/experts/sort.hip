// Tokens' choices sorted by expert (include/experts.h): a stable counting sort.
//
// A workgroup takes a run of choices in order, 64 to a wave at a time. A choice's rank in its wave is the number of lanes
// before it with the same expert, found by ballots on the bits of its number, and the wave's own count of that expert
// so far, which the first such lane then raises. Up to kAlone choices one workgroup does it all. More are runs of kRun, first
// each run's counts, then the ranks; up to kFewRuns runs each adds the counts before it by itself, for more a launch
// between the two makes their prefix sums. No order depends on an atomic.
// Bound by launches and by latency: 96 choices 3.4 us, 6002 8.6 in one launch (three launches of runs: 12), 32,768 12 in two and
// 65,536 15 (three: 17). A choice is 8 bytes in and 8 out.
#include "experts.h"
#include "hip_support.h"
#include "blocks/device_blocks.h"

namespace {

using namespace blocks;

constexpr unsigned kThreads = 1024, kWaves = kThreads / kWave, kTurns = 4, kRun = kThreads * kTurns;
constexpr unsigned kAloneTurns = 16, kAlone = kThreads * kAloneTurns, kFewRuns = 64;

struct Sort {
    const void* ids;
    std::int32_t *offsets, *order, *places;
    std::uint32_t* counts; // [experts + 1][runs], then [experts + 1] totals
    unsigned choices, experts, runs;
};

// The expert of a choice; those of none are one after the last.
template <typename Id> __device__ __forceinline__ unsigned expertOf(const Sort& a, unsigned c) {
    const Id e = static_cast<const Id*>(a.ids)[c];
    return e >= 0 && e < Id(a.experts) ? unsigned(e) : a.experts;
}

template <typename Id> __global__ __launch_bounds__(kThreads) void countChoices(Sort a) {
    extern __shared__ unsigned counts[];
    const unsigned run = blockIdx.x, t = threadIdx.x;
    for (unsigned e = t; e <= a.experts; e += kThreads) counts[e] = 0;
    __syncthreads();
#pragma unroll
    for (unsigned i = 0; i < kTurns; ++i) {
        const std::uint64_t c = std::uint64_t(run) * kRun + i * kThreads + t;
        if (c < a.choices) atomicAdd(&counts[expertOf<Id>(a, unsigned(c))], 1u);
    }
    __syncthreads();
    for (unsigned e = t; e <= a.experts; e += kThreads) a.counts[std::uint64_t(e) * a.runs + run] = counts[e];
}

// The sum of v over the threads before this one, and over all.
__device__ __forceinline__ unsigned scanGroup(unsigned v, unsigned* waves, unsigned& total) {
    const unsigned lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    unsigned upTo = v;
#pragma unroll
    for (unsigned by = 1; by < kWave; by *= 2) {
        const unsigned up = unsigned(__shfl_up(int(upTo), by));
        upTo += lane >= by ? up : 0;
    }
    if (lane == kWave - 1) waves[wave] = upTo;
    __syncthreads();
    unsigned before = 0;
    total = 0;
    for (unsigned w = 0; w < kWaves; ++w) {
        before += w < wave ? waves[w] : 0;
        total += waves[w];
    }
    __syncthreads();
    return before + upTo - v;
}

// One expert's counts become the counts before each run; their total goes behind all counts.
__global__ __launch_bounds__(kThreads) void scanCounts(Sort a) {
    __shared__ unsigned waves[kWaves];
    std::uint32_t* counts = a.counts + std::uint64_t(blockIdx.x) * a.runs;
    unsigned before = 0;
    for (unsigned base = 0; base < a.runs; base += kThreads) {
        const unsigned run = base + threadIdx.x, v = run < a.runs ? counts[run] : 0;
        unsigned total;
        const unsigned at = scanGroup(v, waves, total);
        if (run < a.runs) counts[run] = before + at;
        before += total;
    }
    if (threadIdx.x == 0) a.counts[std::uint64_t(a.experts + 1) * a.runs + blockIdx.x] = before;
}

// Alone: the only run, whose own counts are all there are. Scanned: counts are those before each run.
enum class Counts { alone, each, scanned };
template <typename Id, unsigned Turns, Counts C> __global__ __launch_bounds__(kThreads) void placeChoices(Sort a) {
    extern __shared__ unsigned lds[]; // counts of each wave, [kWaves][experts + 1]; then the first row of each expert
    __shared__ unsigned waves[kWaves];
    const unsigned t = threadIdx.x, lane = t % kWave, wave = t / kWave, run = blockIdx.x, all = a.experts + 1;
    unsigned *counts = lds + wave * all, *starts = lds + kWaves * all;
    for (unsigned i = t; i < kWaves * all; i += kThreads) lds[i] = 0;
    __syncthreads();
    // A wave's choices lie in a row; alone, the waves share what there is.
    const unsigned turns = C == Counts::alone ? (a.choices + kThreads - 1) / kThreads : Turns;
    const std::uint64_t first = std::uint64_t(run) * kRun + wave * turns * kWave + lane;
    unsigned expert[Turns], rank[Turns];
#pragma unroll
    for (unsigned i = 0; i < Turns; ++i) {
        const std::uint64_t c = first + i * kWave;
        expert[i] = i < turns && c < a.choices ? expertOf<Id>(a, unsigned(c)) : ~0u;
    }
    const unsigned bits = 32 - __builtin_clz(a.experts);
#pragma unroll
    for (unsigned i = 0; i < Turns; ++i) {
        if (i >= turns) break;
        const bool in = expert[i] != ~0u;
        std::uint64_t same = __ballot(in);
        for (unsigned b = 0; b < bits; ++b) {
            const std::uint64_t set = __ballot(expert[i] >> b & 1);
            same &= expert[i] >> b & 1 ? set : ~set;
        }
        const unsigned before = __builtin_popcountll(same & ((std::uint64_t(1) << lane) - 1));
        const unsigned so = in ? counts[expert[i]] : 0;
        __builtin_amdgcn_wave_barrier();
        if (in && before == 0) counts[expert[i]] = so + unsigned(__builtin_popcountll(same));
        __builtin_amdgcn_wave_barrier();
        rank[i] = so + before;
    }
    __syncthreads();
    // Counts become the counts before each wave, and starts the first row of each expert of this run.
    unsigned before = 0;
    for (unsigned base = 0; base < all; base += kThreads) {
        const unsigned e = base + t;
        unsigned mine = 0;
        if (e < all)
            for (unsigned w = 0; w < kWaves; ++w) {
                const unsigned n = lds[w * all + e];
                lds[w * all + e] = mine;
                mine += n;
            }
        unsigned earlier = 0; // of this expert, in the runs before
        if (C == Counts::scanned && e < all) {
            mine = a.counts[std::uint64_t(all) * a.runs + e];
            earlier = a.counts[std::uint64_t(e) * a.runs + run];
        }
        if (C == Counts::each && e < all) {
            mine = 0;
            for (unsigned r = 0; r < a.runs; ++r) {
                const unsigned n = a.counts[std::uint64_t(e) * a.runs + r];
                earlier += r < run ? n : 0;
                mine += n;
            }
        }
        unsigned total;
        const unsigned start = before + scanGroup(mine, waves, total);
        before += total;
        if (e < all) {
            starts[e] = start + earlier;
            if (run == 0) a.offsets[e] = std::int32_t(start);
        }
    }
    __syncthreads();
#pragma unroll
    for (unsigned i = 0; i < Turns; ++i) {
        if (expert[i] == ~0u) continue;
        const unsigned c = unsigned(first + i * kWave), row = starts[expert[i]] + counts[expert[i]] + rank[i];
        a.places[c] = std::int32_t(row);
        a.order[row] = std::int32_t(c);
    }
}

std::uint64_t runsOf(std::uint32_t choices) { return (std::uint64_t(choices) + kRun - 1) / kRun; }

} // namespace

std::size_t sortExpertsWorkspace(std::uint32_t choices, std::uint32_t experts) {
    if (choices <= kAlone) return 0;
    return std::size_t((runsOf(choices) + 1) * (std::uint64_t(experts) + 1) * 4 + 255) / 256 * 256;
}

void sortExperts(const void* ids, std::uint32_t idBytes, ExpertPlan plan, void* workspace, std::size_t workspaceBytes,
                 hipStream_t stream) {
    const char* where = "sort experts";
    if (idBytes != 4 && idBytes != 8) reject(where, "choices must be of 4 or 8 bytes");
    if (!plan.experts || plan.experts > kMaxExperts) reject(where, "experts must be 1 to 1024");
    if (plan.choices >> 31) reject(where, "2^31 choices or more");
    if (!plan.offsets || (plan.choices && (!ids || !plan.order || !plan.places))) reject(where, "null choices or plan");
    if (reinterpret_cast<std::uintptr_t>(ids) % idBytes) reject(where, "choices not aligned to their type");
    if ((reinterpret_cast<std::uintptr_t>(plan.offsets) | reinterpret_cast<std::uintptr_t>(plan.order) |
         reinterpret_cast<std::uintptr_t>(plan.places)) % 4)
        reject(where, "plan not aligned to its elements");
    const std::size_t need = sortExpertsWorkspace(plan.choices, plan.experts);
    if (need > workspaceBytes || (need && !workspace)) reject(where, "workspace too small");
    if (reinterpret_cast<std::uintptr_t>(workspace) % 16) reject(where, "workspace must be 16-byte aligned");
    Sort a = {ids, plan.offsets, plan.order, plan.places, static_cast<std::uint32_t*>(workspace), plan.choices, plan.experts,
              unsigned(runsOf(plan.choices))};
    const unsigned all = plan.experts + 1, lds = (kWaves + 1) * all * 4;
    const auto sort = [&](auto id) {
        typedef decltype(id) Id;
        const dim3 one(1), runs(a.runs), threads(kThreads);
        if (plan.choices <= kRun)
            hipLaunchKernelGGL((placeChoices<Id, kTurns, Counts::alone>), one, threads, lds, stream, a);
        else if (!need)
            hipLaunchKernelGGL((placeChoices<Id, kAloneTurns, Counts::alone>), one, threads, lds, stream, a);
        else
            hipLaunchKernelGGL((countChoices<Id>), runs, threads, all * 4, stream, a);
        if (need && a.runs <= kFewRuns)
            hipLaunchKernelGGL((placeChoices<Id, kTurns, Counts::each>), runs, threads, lds, stream, a);
        if (need && a.runs > kFewRuns) {
            hipLaunchKernelGGL(scanCounts, dim3(all), threads, 0, stream, a);
            hipLaunchKernelGGL((placeChoices<Id, kTurns, Counts::scanned>), runs, threads, lds, stream, a);
        }
    };
    if (idBytes == 4)
        sort(std::int32_t{});
    else
        sort(std::int64_t{});
    checkHip(hipGetLastError());
}
