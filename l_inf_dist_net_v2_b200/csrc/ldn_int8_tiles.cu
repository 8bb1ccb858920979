// Which tensor-core kernel an integer product takes, and its launch.
#include "ldn_int8_tiles.cuh"

namespace ldn {
namespace {

// Clusters of CTAs with an SM each that the device holds at the same time: GPCs have different numbers of SMs, so it is not the
// quotient (eight 8s too many took twice the time).
int resident_clusters(int size, const DeviceCtx* ctx) {
    static std::atomic<int> known[64][9];
    const int have = known[ctx->device][size].load(std::memory_order_acquire);
    if (have > 0) return have;
    cudaLaunchAttribute attr[1] = {};
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = size;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctx->sm_count / size * size);
    cfg.blockDim = dim3(kProductThreads);
    cfg.dynamicSmemBytes = pair_smem();
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int count = 0;
    if (allow_smem(product_pairs_kernel<float>, pair_smem()) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&count, product_pairs_kernel<float>, &cfg) != cudaSuccess || count < 1) {
        cudaGetLastError();
        count = ctx->sm_count / size;
    }
    known[ctx->device][size].store(count, std::memory_order_release);
    return count;
}

struct Plan {
    int tokens;  // of a tile; 0: pairs of CTAs
    int ranks;   // CTAs that share a tile's terms
};

// The plan with the smallest estimate, in clocks.  A stage takes as long as its bytes (95 per clock into one SM, 10500 into all),
// its products (two clocks per token, pairs: 512), or a load's way divided by the stages in flight; then there are the start, the
// stores (20 clocks per token, pairs: beside the next tile's products where those take longer) and the way of split sums.
// Measured, 5120 -> 5120, us: 64 tokens, tiles of 64 in 1 / 3 shares 9.4 / 8.8, of 128 10.2; 256 tokens, tiles of 128 11.7, of 256
// 16.5, pairs 17.9; 2048 tokens, tiles of 256 49, pairs 44; 10000 tokens 196, 161.
Plan plan_of(const ProductArgs& a, const DeviceCtx* ctx) {
    const int kt = (a.K + kTerms - 1) / kTerms;
    const long long tiles_n = (a.N + kLanes - 1) / kLanes;
    Plan best = {0, 1};
    const long long pairs = resident_clusters(2, ctx);
    const long long pair_tiles = ((a.N + 2 * kLanes - 1) / (2 * kLanes)) * ((a.M + kPairTokens - 1) / kPairTokens);
    const double pair_tile = kt * 520.0 > 4700.0 ? kt * 520.0 : 4700.0;
    double least = 10000.0 + (pair_tiles + pairs - 1) / pairs * pair_tile + 4700.0;
    for (int tokens = 16; tokens <= 256; tokens *= 2) {
        if (tokens < 256 && a.M > 8 * tokens) continue;
        const long long tiles = tiles_n * ((a.M + tokens - 1) / tokens);
        const double stored = 20.0 * (a.M < tokens ? a.M : tokens);
        for (int ranks = 1; ranks <= (tokens == 256 ? 1 : 8) && ranks <= kt; ++ranks) {
            const long long resident = ranks == 1 ? ctx->sm_count : resident_clusters(ranks, ctx), waves = (tiles + resident - 1) / resident;
            const double at_once = (tiles < resident ? tiles : resident) * ranks, bytes = stage_bytes(tokens);
            double stage = 260.0;
            for (const double t : {bytes / 95.0, bytes * at_once / 10500.0, 2.05 * tokens})
                if (t > stage) stage = t;
            const double cost = 4500.0 + waves * ((kt + ranks - 1) / ranks * stage + 2000.0 +
                                                  (ranks > 1 ? 2000.0 + 15.0 * tokens + stored / ranks : stored));
            if (cost < least) {
                least = cost;
                best = {tokens, ranks};
            }
        }
    }
    return best;
}

template <int TOKENS, class T>
int launch_split(const ProductArgs& a, int ranks, int kt, int* status, cudaStream_t st) {
    CUtensorMap map_w, map_q;
    int r = make_byte_map(&map_w, a.w, a.K, a.N, a.pitch_w, kLanes);
    if (r == kOk) r = make_byte_map(&map_q, a.q, a.K, a.M, a.pitch_q, TOKENS);
    if (r != kOk) return r;
    static OncePerDevice once;
    r = once([] { return allow_smem(product_split_kernel<TOKENS, T>, split_smem(TOKENS)); });
    if (r != kOk) return r;
    const int tiles_n = (a.N + kLanes - 1) / kLanes;
    const unsigned grid = static_cast<unsigned>(tiles_n * ((a.M + TOKENS - 1) / TOKENS) * ranks);
    return launch_after_in_clusters(product_split_kernel<TOKENS, T>, ranks, grid, kProductThreads, split_smem(TOKENS), st, map_w, map_q,
                                    a, tiles_n, kt, status);
}

template <class T>
int launch_pairs(const ProductArgs& a, int kt, int* status, const DeviceCtx* ctx, cudaStream_t st) {
    CUtensorMap map_w, map_q;
    int r = make_byte_map(&map_w, a.w, a.K, a.N, a.pitch_w, kLanes);
    if (r == kOk) r = make_byte_map(&map_q, a.q, a.K, a.M, a.pitch_q, kLanes);
    if (r != kOk) return r;
    static OncePerDevice once;
    r = once([] { return allow_smem(product_pairs_kernel<T>, pair_smem()); });
    if (r != kOk) return r;
    const int tiles_n = (a.N + 2 * kLanes - 1) / (2 * kLanes);
    const long long tiles = tiles_n * ((a.M + kPairTokens - 1) / kPairTokens);
    const long long pairs = resident_clusters(2, ctx);
    return launch_after_in_clusters(product_pairs_kernel<T>, 2, static_cast<unsigned>(2 * (tiles < pairs ? tiles : pairs)),
                                    kProductThreads, pair_smem(), st, map_w, map_q, a, tiles_n, static_cast<int>(tiles), kt, status);
}

}  // namespace

int launch_product_tiles(const ProductArgs& whole, int type, int* status, const DeviceCtx* ctx, cudaStream_t st) {
    const Plan plan = plan_of(whole, ctx);
    const int kt = (whole.K + kTerms - 1) / kTerms;
    // tiles are counted in 32 bits: at most 2^27 of the smallest ones per launch
    const long long tiles_n = (whole.N + kLanes - 1) / kLanes, most = ((1LL << 24) / tiles_n + 1) * 16;
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        for (long long first = 0; first < whole.M;) {
            ProductArgs a = whole;
            const long long chunk = most / 256 * 256 + 256;
            a.M = whole.M - first < chunk ? whole.M - first : chunk;
            a.q += first * a.pitch_q;
            a.scale += first;
            a.out = static_cast<T*>(a.out) + first * a.N;
            int r;
            switch (plan.tokens) {
                case 16: r = launch_split<16, T>(a, plan.ranks, kt, status, st); break;
                case 32: r = launch_split<32, T>(a, plan.ranks, kt, status, st); break;
                case 64: r = launch_split<64, T>(a, plan.ranks, kt, status, st); break;
                case 128: r = launch_split<128, T>(a, plan.ranks, kt, status, st); break;
                case 256: r = launch_split<256, T>(a, plan.ranks, kt, status, st); break;
                default: r = launch_pairs<T>(a, kt, status, ctx, st);
            }
            if (r != kOk) return r;
            first += a.M;
        }
        return static_cast<int>(kOk);
    });
}

}  // namespace ldn
