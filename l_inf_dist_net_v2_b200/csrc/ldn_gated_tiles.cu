// How the tiles of the gated projection's products are dealt out, and their launch.
#include "ldn_gated_tiles.cuh"

namespace ldn {
namespace {

// Pairs of CTAs that the device holds at the same time
int resident_pairs(const DeviceCtx* ctx) {
    static std::atomic<int> known[64];
    const int have = known[ctx->device].load(std::memory_order_acquire);
    if (have > 0) return have;
    constexpr auto kernel = gated_tiles_kernel<__nv_bfloat16, GatedForm::Forward, false>;
    cudaLaunchAttribute attr[1] = {};
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctx->sm_count / 2 * 2);
    cfg.blockDim = dim3(kProductThreads);
    cfg.dynamicSmemBytes = kTileSmem;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int count = 0;
    if (allow_smem(kernel, kTileSmem) != cudaSuccess || cudaOccupancyMaxActiveClusters(&count, kernel, &cfg) != cudaSuccess || count < 1) {
        cudaGetLastError();
        count = ctx->sm_count / 2;
    }
    known[ctx->device].store(count, std::memory_order_release);
    return count;
}

int steps_over(long long n, int size) { return static_cast<int>((n + size - 1) / size); }

// The tiles behind the last whole round are shared out in equal ranges where that saves more than storing and adding up the parts costs
// (both in clocks: a step takes 512, a pair stores and another kernel reads 1 KB per row of a part at 4000 bytes per clock).
void plan(GatedForm form, long long M, int N, int terms, int type, const DeviceCtx* ctx, TileArgs* a) {
    const bool parted = type == LDN_F32;
    a->drained = !parted && static_cast<long long>(terms) * (form == GatedForm::GradRows ? 2 : 1) > kMostTerms;
    const int unit_steps = parted ? kUnitSteps<float, false> : a->drained ? kUnitSteps<__half, true> : 1;
    a->M = M;
    a->N = N;
    a->tiles_m = steps_over(M, kSide);
    a->tiles_n = steps_over(N, form == GatedForm::Forward ? kSide / 2 : kSide);
    a->tiles = a->tiles_m * a->tiles_n * (form == GatedForm::GradWeights ? 2 : 1);
    a->side_steps = steps_over(terms, kStepTerms);
    a->side_units = steps_over(a->side_steps, unit_steps);
    a->units = a->side_units * (form == GatedForm::GradRows ? 2 : 1);
    const long long least = parted || a->drained ? 1 : 4, shares = (static_cast<long long>(a->tiles) * a->units + least - 1) / least;
    const int held = resident_pairs(ctx), resident = held < kMostPairs ? held : kMostPairs;
    // (a tile each at least: 85, 9 -> 7429 bf16 has 59 of one step; by 15 pairs it took 54 us, by 59 21)
    const long long wanted = shares > a->tiles ? shares : a->tiles;
    a->pairs = static_cast<int>(wanted < resident ? wanted : resident);
    const int rest = a->tiles % a->pairs;
    a->whole = a->tiles;
    if (rest) {
        const double tile = static_cast<double>(a->units) * unit_steps * (parted ? 6 : 1) * 512.0;
        const double rows = M < kSide ? static_cast<double>(M) : kSide;
        if (tile * (1.0 - static_cast<double>(rest) / a->pairs) > 5000.0 + (a->pairs + rest) * rows * 2048.0 / 4000.0) a->whole = a->tiles - rest;
        else if (a->tiles < a->pairs) a->pairs = a->tiles;
    }
}
size_t scratch_of(const TileArgs& a) {
    return a.whole < a.tiles ? static_cast<size_t>(2 * a.pairs) * kSide * kSide * sizeof(float) : 0;
}

int map_of(CUtensorMap* map, const Images& o, bool across) {
    return make_image_map(map, o.base, o.columns, o.rows, o.count, o.pitch, o.count > 1 ? o.apart : o.pitch, across ? kStepTerms : 128);
}

template <class T, GatedForm F, bool LONG>
int launch(const TileArgs& a, const CUtensorMap& map_a, const CUtensorMap& map_b0, const CUtensorMap& map_b1, cudaStream_t st) {
    constexpr auto kernel = gated_tiles_kernel<T, F, LONG>;
    static OncePerDevice once;
    int r = once([] { return allow_smem(kernel, kTileSmem); });
    if (r != kOk) return r;
    r = launch_after_in_clusters(kernel, 2, static_cast<unsigned>(2 * a.pairs), kProductThreads, kTileSmem, st, map_a, map_b0, map_b1, a);
    if (r != kOk || a.whole == a.tiles) return r;
    const unsigned rows = a.M < kSide ? static_cast<unsigned>((a.M + kFixRows - 1) / kFixRows) : kSide / kFixRows;
    return launch_after(gated_parts_kernel<T, F>, dim3(a.tiles - a.whole, rows), kFixRows * kFixRuns<F>, 0, st, a);
}

}  // namespace

size_t gated_tiles_scratch(GatedForm form, long long M, int N, int terms, int type, const DeviceCtx* ctx) {
    TileArgs a = {};
    plan(form, M, N, terms, type, ctx, &a);
    return scratch_of(a);
}

int launch_gated_tiles(GatedForm form, TileArgs a, int terms, const Images& op_a, const Images& op_b0, const Images& op_b1, int type,
                       char* scratch, int* status, const DeviceCtx* ctx, cudaStream_t st) {
    plan(form, a.M, a.N, terms, type, ctx, &a);
    a.partials = reinterpret_cast<float*>(scratch);
    a.status = status;
    CUtensorMap map_a, map_b0, map_b1;
    int r = map_of(&map_a, op_a, form == GatedForm::GradWeights);
    if (r == kOk) r = map_of(&map_b0, op_b0, form != GatedForm::Forward);
    if (r == kOk) r = map_of(&map_b1, op_b1, form != GatedForm::Forward);
    if (r != kOk) return r;
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        auto go = [&](auto drained) {
            constexpr bool kLong = decltype(drained)::value;
            switch (form) {
                case GatedForm::Forward: return launch<T, GatedForm::Forward, kLong>(a, map_a, map_b0, map_b1, st);
                case GatedForm::GradRows: return launch<T, GatedForm::GradRows, kLong>(a, map_a, map_b0, map_b1, st);
                default: return launch<T, GatedForm::GradWeights, kLong>(a, map_a, map_b0, map_b1, st);
            }
        };
        if constexpr (!kParted<T>)
            if (a.drained) return go(std::true_type());
        return go(std::false_type());
    });
}

}  // namespace ldn
