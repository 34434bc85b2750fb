// Entry points of the operators around the experts' GEMMs: FP8 GEMMs and quantisers with an FP32 scale per block of 128, the sort of tokens by
// expert with its way back and gradients, SwiGLU with its gradient. Included by dgb200.cu, whose launch helpers and tuning
// knobs it uses.
#pragma once

namespace dgb {
namespace {

// Rows and columns a call may have: tiles and vectors are counted in 32 bits, with room for the last one.
constexpr int kMaxRows = 0x7ffff000, kMaxColumns = 1 << 28;

inline bool aligned_to(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % static_cast<uintptr_t>(bytes) == 0; }

// Raises a kernel's shared-memory limit once per device.
template <typename Kernel>
int allow_dynamic_smem(Kernel kernel, int bytes, std::atomic<int> (&done)[64]) {
    int dev = 0;
    DGB_CUDA(cudaGetDevice(&dev));
    DGB_REQUIRE(dev >= 0 && dev < 64, "device index %d out of range", dev);
    if (done[dev].load(std::memory_order_acquire) == 0) {
        DGB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
        done[dev].store(1, std::memory_order_release);
    }
    return 0;
}

int make_tensor_map_3d_bytes(CUtensorMap* out, const void* base, uint64_t inner, uint64_t rows, uint64_t groups, uint32_t box_rows) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (fn == nullptr) return fail(DGB200_ECUDA, "cuTensorMapEncodeTiled is not available from the CUDA driver");
    const cuuint64_t dims[3] = {inner, rows, groups};
    const cuuint64_t strides[2] = {inner, inner * rows};
    const cuuint32_t box[3] = {128, box_rows, 1};
    const cuuint32_t elem_strides[3] = {1, 1, 1};
    const CUresult r = fn(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, elem_strides,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return fail(DGB200_ECUDA, "cuTensorMapEncodeTiled failed with CUresult %d (%llu x %llu x %llu bytes, box of %u rows)",
                    static_cast<int>(r), static_cast<unsigned long long>(groups), static_cast<unsigned long long>(rows),
                    static_cast<unsigned long long>(inner), box_rows);
    return 0;
}

template <int BLOCK_N, int kStages, bool kF32, bool kPair>
int launch_block_scaled(const CUtensorMap& tm_a, const CUtensorMap& tm_b, const BlockScaledParams& p, int grid, cudaStream_t stream) {
    using L = BlockScaledSmem<BLOCK_N, kStages, kPair>;
    auto kernel = dgb200_block_scaled_gemm_kernel<BLOCK_N, kStages, kF32, kPair>;
    static std::atomic<int> done[64] = {};
    if (const int rc = allow_dynamic_smem(kernel, L::kDynamicBytes, done)) return rc;
    DGB_CUDA(launch_kernel_in_clusters(kPair ? 2 : 1, kernel, dim3(grid), dim3(kGemmThreads), L::kDynamicBytes, stream, use_pdl(), tm_a, tm_b, p));
    return 0;
}

// The split-K form: clusters of `split` CTAs, one for each of `tiles` tiles. `max_clusters` receives how many of them the device runs at
// the same time (asked once per form, size and device; with `dry` nothing is launched).
template <bool kF32>
int launch_block_scaled_split(const CUtensorMap& tm_a, const CUtensorMap& tm_b, const BlockScaledParams& p, int tiles, int split, bool dry,
                              int* max_clusters, cudaStream_t stream) {
    using L = BlockScaledSmem<128, 6, false>;
    auto kernel = dgb200_block_scaled_gemm_kernel<128, 6, kF32, false, true>;
    static std::atomic<int> done[64] = {}, active[64][4] = {};  // [device][log2 split]; 0 = not asked yet
    if (const int rc = allow_dynamic_smem(kernel, L::kDynamicBytes, done)) return rc;
    int dev = 0;
    DGB_CUDA(cudaGetDevice(&dev));
    std::atomic<int>& known = active[dev][split == 2 ? 1 : (split == 4 ? 2 : 3)];
    int clusters = known.load(std::memory_order_acquire);
    if (clusters == 0) {
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(static_cast<unsigned>(split));
        cfg.blockDim = dim3(kGemmThreads);
        cfg.dynamicSmemBytes = L::kDynamicBytes;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = static_cast<unsigned>(split);
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        DGB_CUDA(cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg));
        known.store(clusters > 0 ? clusters : -1, std::memory_order_release);
    }
    *max_clusters = std::max(clusters, 0);
    if (dry) return 0;
    DGB_CUDA(launch_kernel_in_clusters(split, kernel, dim3(static_cast<unsigned>(tiles * split)), dim3(kGemmThreads), L::kDynamicBytes, stream,
                                       use_pdl(), tm_a, tm_b, p));
    return 0;
}

// CTAs per tile of a dense GEMM (1: no split): the largest of 8, 4 and 2 for which all clusters run at once and every part gets at least three
// groups of kScaleKb K blocks, 12 or, where the last group is short, 9. Device time of calls back to back, no split -> split (us): 7 x 4096 x 7168 15.7 -> 11.0 (4), 33 x 1536 x 7168 15.1 -> 10.5
// (4; 8: 11.1), 512 x 2112 x 7168 16.3 -> 15.4 (2), 128 x 7168 x 16384 35.1 -> 29.4 (2). With less K it does not pay: 1 x 7168 x 2048 7.2 -> 7.8
// (2), 64 x 7168 x 2048 7.5 -> 9.3 (2), 128 x 4096 x 2048 7.0 -> 9.6 (2).
int block_scaled_split(long long tiles, int num_kb, bool f32, int sms, int* split) {
    *split = 1;
    if (tuning().split_k == 0) return 0;
    const int units = (num_kb + kScaleKb - 1) / kScaleKb;
    for (const int s : {8, 4, 2}) {
        if (tuning().split_k > 0 ? s != tuning().split_k || units < s : units < 3 * s) continue;
        if (tiles * s > sms) continue;
        int clusters = 0;
        const CUtensorMap none{};
        const int rc = f32 ? launch_block_scaled_split<true>(none, none, BlockScaledParams{}, 0, s, true, &clusters, nullptr)
                           : launch_block_scaled_split<false>(none, none, BlockScaledParams{}, 0, s, true, &clusters, nullptr);
        if (rc) return rc;
        if (tiles > clusters) continue;
        *split = s;
        return 0;
    }
    return 0;
}

int run_block_scaled_gemm(const dgb200_fp8_block_scaled_gemm_args& a, cudaStream_t stream) {
    const bool dense = a.layout_kind == DGB200_LAYOUT_DENSE, masked = a.layout_kind == DGB200_LAYOUT_MASKED;
    const bool row_ids = a.layout_kind == DGB200_LAYOUT_ROW_IDS, psum = a.layout_kind == DGB200_LAYOUT_PSUM;
    DGB_REQUIRE(dense || masked || row_ids || psum, "unknown layout kind %d", a.layout_kind);
    DGB_REQUIRE(a.m >= 0 && a.n > 0 && a.k > 0 && a.num_groups > 0, "m must be >= 0, n, k and num_groups positive");
    DGB_REQUIRE(a.m <= kMaxRows && a.n <= kMaxColumns && a.k <= kMaxColumns, "m (%d), n (%d) or k (%d) is too large", a.m, a.n, a.k);
    DGB_REQUIRE(a.n % 8 == 0 && a.k % 16 == 0, "n (%d) must be a multiple of 8 and k (%d) of 16", a.n, a.k);
    DGB_REQUIRE(!a.b_mn_major || a.n % 16 == 0, "an MN-major b needs n (%d) to be a multiple of 16", a.n);
    DGB_REQUIRE(!dense || a.num_groups == 1, "the dense form has one group");
    DGB_REQUIRE((!psum && !masked) || a.num_groups <= kMaxCachedGroups, "at most %d groups", kMaxCachedGroups);
    DGB_REQUIRE(!psum || (a.alignment > 0 && a.alignment % 4 == 0), "alignment (%d) must be a positive multiple of 4", a.alignment);
    DGB_REQUIRE(!row_ids || (a.alignment > 0 && a.alignment % 128 == 0),
                "the row-id layout needs an M alignment that is a multiple of 128, got %d", a.alignment);
    if (a.m == 0) return 0;
    DGB_REQUIRE(a.a != nullptr && a.sfa != nullptr && a.b != nullptr && a.sfb != nullptr && a.d != nullptr && (dense || a.layout != nullptr),
                "null tensor pointer");
    DGB_REQUIRE(aligned_to(a.a, 16) && aligned_to(a.b, 16), "a and b must be 16-byte aligned");
    DGB_REQUIRE(aligned_to(a.sfa, 4) && aligned_to(a.sfb, 4) && aligned_to(a.layout, 4), "scales and layout must be 4-byte aligned");
    const int out_bytes = a.d_is_fp32 ? 4 : 2;
    DGB_REQUIRE(aligned_to(a.d, 16), "d must be 16-byte aligned");
    DGB_REQUIRE(a.d_row_stride >= a.n && (a.d_row_stride * out_bytes) % 16 == 0, "d row stride must cover n and keep rows 16-byte aligned");
    DGB_REQUIRE(a.c == nullptr || (dense && a.d_is_fp32), "c needs the dense form and a float32 d");
    DGB_REQUIRE(a.c == nullptr || (aligned_to(a.c, 16) && a.c_row_stride >= a.n && a.c_row_stride % 4 == 0),
                "c must be 16-byte aligned with rows that cover n");
    BlockScaledParams p{};
    p.sfa = a.sfa;
    p.sfb = a.sfb;
    p.sfa_group_stride = a.sfa_group_stride;
    p.sfa_row_stride = a.sfa_row_stride;
    p.sfa_k_stride = a.sfa_k_stride;
    p.sfb_group_stride = a.sfb_group_stride;
    p.sfb_n_stride = a.sfb_n_stride;
    p.sfb_k_stride = a.sfb_k_stride;
    p.d = a.d;
    p.c = a.c;
    p.d_row_stride = a.d_row_stride;
    p.c_row_stride = a.c_row_stride;
    p.layout = a.layout;
    p.mode = dense ? kModeDense : (masked ? kModeMasked : (psum ? kModePsum : kModeRowIds));
    p.m = a.m;
    p.n = a.n;
    p.k = a.k;
    p.num_groups = a.num_groups;
    p.alignment = dense || masked ? 128 : a.alignment;
    p.store_padding = psum && a.store_padding;
    p.b_mn_major = a.b_mn_major ? 1 : 0;
    p.sf_vec = a.sfa_k_stride == 1 && aligned_to(a.sfa, 16) && a.sfa_row_stride % 4 == 0 && a.sfa_group_stride % 4 == 0;
    int sms = 0;
    if (const int rc = effective_num_sms(&sms)) return rc;

    // Tiles of 128 rows that the call may have. Masked and psum: the host knows the buffer, not the rows in use.
    const long long groups = dense || row_ids ? 1 : a.num_groups;
    const long long expected = masked ? std::min<long long>(std::max(a.expected_m, 1), a.m) : (psum ? (a.m + groups - 1) / groups : a.m);
    const long long m_tiles = groups * ((expected + 127) / 128);
    auto tiles_at = [&](int bn) { return m_tiles * ((a.n + bn - 1) / bn); };
    // The tile width whose waves take the least time: a K block of a 256-, 128-, 64- or 32-wide tile takes about 540, 310, 260 or 240 ns, the
    // narrow ones because a K block has fixed costs. 1999 x 2112 x 7168 (FP32, accumulated): 144 tiles of 256 52 us, 272 of 128 56.
    // Groups of few rows read their weights at HBM rate, and tiles of 128 leave a shorter last wave: 32 groups of 24 rows, 256 -> 128 wide:
    // N 7168, K 2048 89 -> 84 us, N 4096, K 7168 161 -> 154; 64 of 8 rows, N 4096, K 4096 169 -> 171. Tile width and loads of 32 rows (below)
    // together, masked buffers of 256 rows, 32 groups, without -> with: N 4096, K 7168 8 rows 165 -> 152, 24 174 -> 152, 48 179 -> 162, 96
    // 183 -> 175; N 7168, K 2048 48 rows 99 -> 86, 96 102 -> 92. Past the bound it would still serve one tile of rows (112 rows 184 -> 173 and
    // 107 -> 96, 128 rows 183 -> 177 and 106 -> 103) and lose with two (160 rows 316 -> 340 and 149 -> 176, 192 rows 309 -> 357).
    // With psum the host knows the buffer's rows only: a plan's buffer of alignment 128 is not taken for one of few rows.
    const bool few_rows = (masked || psum) && expected <= 96;
    int block_n = 256;
    if (tuning().block_n != 0) {
        block_n = tuning().block_n;
    } else {
        long long best = -1;
        constexpr int kWidths[4] = {256, 128, 64, 32}, kCost[4] = {54, 31, 26, 24};
        for (int i = few_rows ? 1 : 0; i < (a.b_mn_major ? 2 : 4); ++i) {
            const long long cost = (tiles_at(kWidths[i]) + sms - 1) / sms * kCost[i];
            if (best < 0 || cost < best) {
                best = cost;
                block_n = kWidths[i];
            }
        }
    }
    int split = 1;
    if (dense && tuning().block_n == 0) {
        if (const int rc = block_scaled_split(tiles_at(128), (a.k + 127) / 128, a.d_is_fp32 != 0, sms, &split)) return rc;
        if (split > 1) block_n = 128;
    }
    // Pairs load 32 KB per SM and K block instead of 48. Single CTAs -> pairs (us): dense 4096 x 4096 x 7168 116 -> 111, 8192 x 7168 x 4096
    // 228 -> 216. With groups half a pair tile is lost on every second one: N 4096, K 7168, 32 groups of 247 rows 323 -> 371, 8 of
    // 900 239 -> 250. Above the bound, in turn, 4 groups: N 4096, K 7168 2100 rows 286 -> 284, 2500 333 -> 321, 4000 508 -> 488, 6000 737 ->
    // 712; N 7168, K 2048 170 -> 178, 166 -> 159, 292 -> 284, 433 -> 431 (2100 rows are 17 tiles of 128 but 9 of 256). Below it groups that
    // fill their last pair tile would gain as much (1000, 1500, 2000 rows: 2 to 4 %), but the host does not know the groups.
    const long long pair_tiles = groups * ((expected + 255) / 256) * ((a.n + 255) / 256);
    const bool pair = !row_ids && block_n == 256 && sms >= 2 && tuning().pair != 0 &&
                      (tuning().pair == 1 || (expected > (dense ? 128 : 2048) && pair_tiles * 2 >= sms));
    p.a_box_rows = 128;
    if (!pair && (dense || masked) && a.m < 128) p.a_box_rows = (a.m + 7) / 8 * 8;
    // Groups of few rows: 32 at a time, as many as the tile has; a 128-row load would bring the other rows of the buffer as well
    // (32 groups of 24 rows, N 4096, K 7168: 163 -> 154 us; 64 of 8, N 4096, K 4096: 176 -> 169).
    if (!pair && few_rows) p.a_box_rows = std::min(p.a_box_rows, 32);

    CUtensorMap tm_a, tm_b;
    int rc = make_tensor_map_3d_bytes(&tm_a, a.a, static_cast<uint64_t>(a.k), static_cast<uint64_t>(a.m), masked ? a.num_groups : 1,
                                      static_cast<uint32_t>(p.a_box_rows));
    if (rc) return rc;
    const int channels = pair ? 128 : block_n;  // of B that one load brings
    rc = a.b_mn_major ? make_tensor_map_3d_bytes(&tm_b, a.b, static_cast<uint64_t>(a.n), static_cast<uint64_t>(a.k), a.num_groups, 128)
                      : make_tensor_map_3d_bytes(&tm_b, a.b, static_cast<uint64_t>(a.k), static_cast<uint64_t>(a.n), a.num_groups,
                                                 static_cast<uint32_t>(channels));
    if (rc) return rc;
    // upper bound of the tiles: a group may end in a short one
    const long long max_tiles = ((masked ? groups * ((a.m + 127ll) / 128) : (a.m + 127ll) / 128 + (psum ? groups : 0))) * ((a.n + block_n - 1) / block_n);
    DGB_REQUIRE(max_tiles < (1ll << 31), "too many output tiles");
    if (split > 1) {
        int clusters = 0;
        const int tiles = static_cast<int>(tiles_at(128));
        return a.d_is_fp32 ? launch_block_scaled_split<true>(tm_a, tm_b, p, tiles, split, false, &clusters, stream)
                           : launch_block_scaled_split<false>(tm_a, tm_b, p, tiles, split, false, &clusters, stream);
    }
    int grid = static_cast<int>(std::min<long long>(sms, max_tiles));
    if (pair) grid = std::max(2, std::min(sms / 2 * 2, static_cast<int>((max_tiles + 1) / 2 * 2)));
#define DGB_BS_LAUNCH(BN, STAGES, PAIR)                                                            \
    return a.d_is_fp32 ? launch_block_scaled<BN, STAGES, true, PAIR>(tm_a, tm_b, p, grid, stream) \
                       : launch_block_scaled<BN, STAGES, false, PAIR>(tm_a, tm_b, p, grid, stream)
    if (pair) DGB_BS_LAUNCH(256, 6, true);
    switch (block_n) {
        case 256: DGB_BS_LAUNCH(256, 4, false);
        case 128: DGB_BS_LAUNCH(128, 6, false);
        case 64: DGB_BS_LAUNCH(64, 8, false);
        default: DGB_BS_LAUNCH(32, 8, false);
    }
#undef DGB_BS_LAUNCH
}

int check_cast_f32(const void* x, const void* q, const float* sf, int rows, int k, long long x_row_stride, long long q_row_stride) {
    DGB_REQUIRE(rows >= 0 && k > 0 && k % 16 == 0, "k (%d) must be a positive multiple of 16", k);
    DGB_REQUIRE(rows <= kMaxRows && k <= kMaxColumns, "rows (%d) or k (%d) too large", rows, k);
    DGB_REQUIRE(rows == 0 || (x != nullptr && q != nullptr && sf != nullptr), "null tensor pointer");
    DGB_REQUIRE(aligned_to(x, 16) && aligned_to(q, 16) && aligned_to(sf, 4) && x_row_stride % 8 == 0 && q_row_stride % 16 == 0,
                "rows of x and q must be 16-byte aligned");
    DGB_REQUIRE(rows <= 1 || (x_row_stride >= k && q_row_stride >= k), "row strides must cover k");
    return 0;
}

constexpr int kMaxSortChunks = 128;

// Entries per chunk of the sort: one CTA counts up to 4096 entries by itself; beyond, chunks of whole 1024s, at most kMaxSortChunks.
int sort_chunk_entries(long long entries) {
    if (entries <= 4096) return 4096;
    return static_cast<int>((entries + 1024ll * kMaxSortChunks - 1) / (1024ll * kMaxSortChunks) * 1024);
}

int vec_bytes_for(std::initializer_list<long long> sizes) {
    long long all = 16;
    for (const long long s : sizes) all |= s;
    return static_cast<int>(all & -all);  // largest power of two up to 16 that divides them all
}

int check_plan(const int32_t* dest_row, const int32_t* expert_end, int tokens, int topk, int experts, int alignment, int capacity) {
    DGB_REQUIRE(tokens >= 0 && topk >= 1 && topk <= 32, "num_topk (%d) must be in [1, 32]", topk);
    DGB_REQUIRE(experts >= 1 && experts <= kMaxPlanExperts, "experts (%d) must be in [1, %d]", experts, kMaxPlanExperts);
    DGB_REQUIRE(alignment >= 1 && capacity >= 0, "alignment must be positive");
    DGB_REQUIRE(alignment <= kMaxColumns, "alignment (%d) is too large", alignment);
    DGB_REQUIRE((dest_row != nullptr || tokens == 0) && expert_end != nullptr, "null tensor pointer");
    return 0;
}

// Columns per CTA: enough CTAs for the machine where there are few tokens.
int column_blocks(int tokens, long long vecs, int threads, int sms) {
    const long long most = (vecs + threads - 1) / threads;
    return static_cast<int>(std::max<long long>(1, std::min<long long>(most, (2ll * sms + tokens - 1) / std::max(tokens, 1))));
}

template <typename Vec, typename ScaleVec>
int launch_permute(const PermuteParams& p, dim3 grid, cudaStream_t stream) {
    DGB_CUDA(launch_kernel(dgb200_permute_kernel<Vec, ScaleVec>, grid, dim3(256), 0, stream, use_pdl(), p));
    return 0;
}

template <typename T>
int launch_unpermute(const UnpermuteParams& p, bool backward, bool wide, dim3 grid, cudaStream_t stream) {
    constexpr int kVec = 16 / sizeof(T);
    if (backward)
        DGB_CUDA(launch_kernel(wide ? dgb200_unpermute_backward_kernel<T, kVec> : dgb200_unpermute_backward_kernel<T, 1>, grid, dim3(256), 0,
                               stream, use_pdl(), p));
    else
        DGB_CUDA(launch_kernel(wide ? dgb200_unpermute_kernel<T, kVec> : dgb200_unpermute_kernel<T, 1>, grid, dim3(128), 0, stream, use_pdl(), p));
    return 0;
}

int run_unpermute(UnpermuteParams& p, bool backward, int is_fp32, cudaStream_t stream) {
    if (const int rc = check_plan(p.dest_row, p.expert_end != nullptr || backward ? p.expert_end : p.dest_row, p.tokens, p.topk, p.experts, p.alignment,
                                  p.capacity))
        return rc;
    DGB_REQUIRE(p.hidden >= 1 && p.hidden <= kMaxColumns, "hidden (%d) must be in [1, %d]", p.hidden, kMaxColumns);
    const int es = is_fp32 ? 4 : 2;
    DGB_REQUIRE(p.out != nullptr || (backward ? p.capacity : p.tokens) == 0, "null output");
    DGB_REQUIRE(p.rows != nullptr || p.capacity == 0, "null tensor pointer");
    DGB_REQUIRE(p.rows_stride >= p.hidden && p.out_stride >= p.hidden && (!backward || p.dy_stride >= p.hidden), "row strides must cover hidden");
    DGB_REQUIRE(!backward || p.tokens == 0 || (p.dy != nullptr && p.d_weights != nullptr), "null tensor pointer");
    DGB_REQUIRE(aligned_to(p.rows, es) && aligned_to(p.out, es) && aligned_to(p.dy, es), "tensors must be aligned to their elements");
    const bool wide = vec_bytes_for({static_cast<long long>(p.hidden) * es, p.rows_stride * es, p.out_stride * es, p.dy_stride * es,
                                     static_cast<long long>(reinterpret_cast<uintptr_t>(p.rows) & 15), static_cast<long long>(reinterpret_cast<uintptr_t>(p.out) & 15),
                                     static_cast<long long>(reinterpret_cast<uintptr_t>(p.dy) & 15)}) == 16;
    dim3 grid(static_cast<unsigned>(p.tokens));
    if (backward) {
        p.padding_blocks = (p.alignment - 1 + 7) / 8;
        const long long blocks = p.tokens + static_cast<long long>(p.experts) * p.padding_blocks;
        DGB_REQUIRE(blocks < (1ll << 31), "too many rows");
        grid.x = static_cast<unsigned>(blocks);
    } else {
        int sms = 0;
        if (const int rc = effective_num_sms(&sms)) return rc;
        const int per = wide ? 16 / es : 1;
        grid.y = static_cast<unsigned>(column_blocks(p.tokens, (p.hidden + per - 1) / per, 128, sms));
    }
    if (grid.x == 0) return 0;
    return is_fp32 ? launch_unpermute<float>(p, backward, wide, grid, stream) : launch_unpermute<__nv_bfloat16>(p, backward, wide, grid, stream);
}

int check_swiglu(const SwigluParams& p, bool backward, int out_width, int out_es) {
    DGB_REQUIRE(p.rows >= 0 && p.inter >= 1, "rows must be >= 0 and inter positive");
    DGB_REQUIRE(p.rows <= kMaxRows && p.inter <= kMaxColumns, "rows (%d) or inter (%d) too large", p.rows, p.inter);
    DGB_REQUIRE(p.rows == 0 || (p.x != nullptr && p.out != nullptr && (!backward || p.dy != nullptr)), "null tensor pointer");
    DGB_REQUIRE(p.layout == nullptr || (p.num_groups > 0 && p.alignment > 0), "a layout needs its groups and alignment");
    DGB_REQUIRE(p.x_stride >= 2ll * p.inter && p.out_stride >= out_width && (!backward || p.dy_stride >= p.inter), "row strides must cover the rows");
    DGB_REQUIRE(aligned_to(p.x, 2) && aligned_to(p.dy, 2) && aligned_to(p.out, out_es), "tensors must be aligned to their elements");
    return 0;
}

constexpr int kSwigluRows = 4;

// A thread per vector of the row, in CTAs no wider than the row. Returns the rows a thread takes: four, so that 8 (backward 12) loads are in
// flight, where that leaves CTAs enough, else one. Backward 36864 x 2 x 2048 with its forward: one row a thread 211 us, two 195, four 181.
int swiglu_launch_shape(int rows, long long vecs, int sms, dim3* grid, dim3* block) {
    const long long blocks = (vecs + 255) / 256;
    const long long threads = ((vecs + blocks - 1) / blocks + 31) / 32 * 32;
    const long long columns = (vecs + threads - 1) / threads;
    const int per_thread = (rows + kSwigluRows - 1) / kSwigluRows * columns * threads >= sms * 1024ll ? kSwigluRows : 1;
    *grid = dim3(static_cast<unsigned>((rows + per_thread - 1) / per_thread), static_cast<unsigned>(columns));
    *block = dim3(static_cast<unsigned>(threads));
    return per_thread;
}

int run_swiglu(const SwigluParams& p, bool backward, cudaStream_t stream) {
    if (const int rc = check_swiglu(p, backward, backward ? 2 * p.inter : p.inter, 2)) return rc;
    if (p.rows == 0) return 0;
    const bool wide = p.inter % 8 == 0 && p.x_stride % 8 == 0 && p.out_stride % 8 == 0 && (!backward || p.dy_stride % 8 == 0) &&
                      aligned_to(p.x, 16) && aligned_to(p.out, 16) && aligned_to(p.dy, 16);
    dim3 grid, block;
    int sms = 0;
    if (const int rc = effective_num_sms(&sms)) return rc;
    const bool many = swiglu_launch_shape(p.rows, wide ? p.inter / 8 : p.inter, sms, &grid, &block) == kSwigluRows;
    DGB_REQUIRE(grid.y <= 65535u, "inter (%d) is too large", p.inter);
    auto kernel = backward ? (wide ? (many ? dgb200_swiglu_backward_kernel<8, kSwigluRows> : dgb200_swiglu_backward_kernel<8, 1>)
                                   : (many ? dgb200_swiglu_backward_kernel<1, kSwigluRows> : dgb200_swiglu_backward_kernel<1, 1>))
                           : (wide ? (many ? dgb200_swiglu_kernel<8, kSwigluRows> : dgb200_swiglu_kernel<8, 1>)
                                   : (many ? dgb200_swiglu_kernel<1, kSwigluRows> : dgb200_swiglu_kernel<1, 1>));
    DGB_CUDA(launch_kernel(kernel, grid, block, 0, stream, use_pdl(), p));
    return 0;
}

}  // namespace
}  // namespace dgb

extern "C" {

using namespace dgb;

int dgb200_fp8_block_scaled_gemm(const dgb200_fp8_block_scaled_gemm_args* args, void* stream) {
    DGB_REQUIRE(args != nullptr && args->struct_size == sizeof(dgb200_fp8_block_scaled_gemm_args), "argument struct of another size");
    return run_block_scaled_gemm(*args, static_cast<cudaStream_t>(stream));
}

int dgb200_per_token_cast_to_fp8_f32_scales(const void* x, int64_t x_row_stride, int32_t rows, int32_t k, int32_t gran_k, void* q,
                                            int64_t q_row_stride, float* sf, int64_t sf_row_stride, void* stream_) {
    if (const int rc = check_cast_f32(x, q, sf, rows, k, x_row_stride, q_row_stride)) return rc;
    DGB_REQUIRE(gran_k == 32 || gran_k == 128, "gran_k must be 32 or 128, got %d", gran_k);
    DGB_REQUIRE(sf_row_stride >= (k + gran_k - 1) / gran_k, "scale rows must hold one scale per gran_k values");
    if (rows == 0) return 0;
    CastF32Params p{};
    p.x = static_cast<const __nv_bfloat16*>(x);
    p.q = static_cast<unsigned char*>(q);
    p.sf = sf;
    p.x_row_stride = x_row_stride;
    p.q_row_stride = q_row_stride;
    p.sf_row_stride = sf_row_stride;
    p.rows = rows;
    p.k = k;
    p.gran_k = gran_k;
    const unsigned columns = static_cast<unsigned>((k + 511) / 512);
    DGB_REQUIRE(columns <= 65535u, "k (%d) is too large", k);
    int sms = 0;
    if (const int rc = effective_num_sms(&sms)) return rc;
    // four rows a warp keep 64 bytes a lane in flight; where that would leave SMs without a CTA, one row
    const bool few = static_cast<long long>((rows + 31) / 32) * columns < 2 * sms;
    const dim3 grid(static_cast<unsigned>(few ? (rows + 7) / 8 : (rows + 31) / 32), columns);
    auto kernel = few ? dgb200_cast_rows_f32_kernel<1, false>
                      : (gran_k == 128 ? dgb200_cast_rows_f32_kernel<4, true> : dgb200_cast_rows_f32_kernel<4, false>);
    DGB_CUDA(launch_kernel(kernel, grid, dim3(256), 0, static_cast<cudaStream_t>(stream_), use_pdl(), p));
    return 0;
}

int dgb200_per_block_cast_to_fp8(const void* x, int64_t x_group_stride, int64_t x_row_stride, int32_t num_groups, int32_t rows, int32_t k,
                                 int32_t use_ue8m0, void* q, int64_t q_group_stride, int64_t q_row_stride, float* sf, int64_t sf_group_stride,
                                 int64_t sf_row_stride, void* stream_) {
    if (const int rc = check_cast_f32(x, q, sf, rows, k, x_row_stride, q_row_stride)) return rc;
    DGB_REQUIRE(num_groups >= 0 && num_groups <= 65535, "at most 65535 groups");
    DGB_REQUIRE(x_group_stride % 8 == 0 && q_group_stride % 16 == 0, "groups of x and q must be 16-byte aligned");
    DGB_REQUIRE(sf_row_stride >= (k + 127) / 128, "scale rows must hold one scale per 128 values");
    DGB_REQUIRE((rows + 127ll) / 128 <= 65535, "rows (%d) are too many", rows);
    if (rows == 0 || num_groups == 0) return 0;
    CastF32Params p{};
    p.x = static_cast<const __nv_bfloat16*>(x);
    p.q = static_cast<unsigned char*>(q);
    p.sf = sf;
    p.x_group_stride = x_group_stride;
    p.x_row_stride = x_row_stride;
    p.q_group_stride = q_group_stride;
    p.q_row_stride = q_row_stride;
    p.sf_group_stride = sf_group_stride;
    p.sf_row_stride = sf_row_stride;
    p.rows = rows;
    p.k = k;
    p.gran_k = 128;
    p.ue8m0 = use_ue8m0 ? 1 : 0;
    const dim3 grid(static_cast<unsigned>((k + 127) / 128), static_cast<unsigned>((rows + 127) / 128), static_cast<unsigned>(num_groups));
    DGB_CUDA(launch_kernel(dgb200_cast_blocks_f32_kernel, grid, dim3(256), 0, static_cast<cudaStream_t>(stream_), use_pdl(), p));
    return 0;
}

int64_t dgb200_moe_dispatch_plan_workspace_bytes(int32_t num_tokens, int32_t num_topk, int32_t num_experts) {
    if (num_tokens < 0 || num_topk < 1 || num_experts < 1) return -1;
    const long long entries = static_cast<long long>(num_tokens) * num_topk;
    const long long chunk = sort_chunk_entries(entries);
    const long long chunks = (entries + chunk - 1) / chunk;
    return chunks <= 1 ? 0 : chunks * num_experts * 4;
}

int dgb200_moe_dispatch_plan(const int64_t* topk_idx, int32_t num_tokens, int32_t num_topk, int32_t num_experts, int32_t alignment,
                             int32_t* dest_row, int32_t* expert_start, int32_t* expert_end, void* workspace, void* stream_) {
    if (const int rc = check_plan(dest_row, expert_end, num_tokens, num_topk, num_experts, alignment, 0)) return rc;
    const long long entries = static_cast<long long>(num_tokens) * num_topk;
    DGB_REQUIRE((topk_idx != nullptr || entries == 0) && expert_start != nullptr, "null tensor pointer");
    DGB_REQUIRE(entries + static_cast<long long>(num_experts) * (alignment - 1) <= kMaxRows, "too many rows");
    const int chunk = sort_chunk_entries(entries);
    const int chunks = static_cast<int>((entries + chunk - 1) / chunk);
    // the kernels form the end of a chunk in 32 bits: above 0x7ffe0000 entries the last one's would be 2^31
    DGB_REQUIRE(static_cast<long long>(chunks) * chunk < (1ll << 31), "too many entries");
    DGB_REQUIRE(chunks <= 1 || (workspace != nullptr && aligned_to(workspace, 4)), "the plan needs its workspace");
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    if (entries <= kPlanThreads) {
        const int threads = std::max<int>(32, (std::max<int>(static_cast<int>(entries), num_experts) + 31) / 32 * 32);
        const size_t smem = static_cast<size_t>((entries + 31) / 32) * ((num_experts + 3) / 4 * 4);
        DGB_CUDA(launch_kernel(dgb200_sort_small_kernel, dim3(1), dim3(threads), smem, stream, use_pdl(), reinterpret_cast<const long long*>(topk_idx),
                               static_cast<int>(entries), num_experts, alignment, dest_row, expert_start, expert_end));
        return 0;
    }
    int* hist = chunks > 1 ? static_cast<int*>(workspace) : nullptr;
    const long long* idx = reinterpret_cast<const long long*>(topk_idx);
    if (hist != nullptr)
        DGB_CUDA(launch_kernel(dgb200_sort_count_kernel, dim3(chunks), dim3(kPlanThreads), 0, stream, use_pdl(), idx, static_cast<int>(entries), chunk,
                               num_experts, hist));
    DGB_CUDA(launch_kernel(dgb200_sort_assign_kernel, dim3(std::max(chunks, 1)), dim3(kPlanThreads), static_cast<size_t>(num_experts) * 32, stream, use_pdl(),
                           idx, static_cast<int>(entries), chunk, num_experts, alignment, static_cast<const int*>(hist), dest_row, expert_start, expert_end));
    return 0;
}

int dgb200_moe_permute(const void* x, int64_t x_row_bytes, int64_t x_row_stride_bytes, void* rows, int64_t rows_row_stride_bytes, const float* x_sf,
                       int32_t sf_per_row, int64_t x_sf_row_stride, float* rows_sf, int64_t rows_sf_row_stride, const int32_t* dest_row,
                       const int32_t* expert_end, int32_t num_tokens, int32_t num_topk, int32_t num_experts, int32_t alignment, int32_t capacity,
                       int32_t zero_padding, void* stream_) {
    if (const int rc = check_plan(dest_row, expert_end, num_tokens, num_topk, num_experts, alignment, capacity)) return rc;
    DGB_REQUIRE(x_row_bytes >= 1 && x_row_stride_bytes >= x_row_bytes && rows_row_stride_bytes >= x_row_bytes, "row strides must cover the rows");
    DGB_REQUIRE((x != nullptr || num_tokens == 0) && (rows != nullptr || capacity == 0), "null tensor pointer");
    DGB_REQUIRE((x_sf == nullptr) == (rows_sf == nullptr) || num_tokens == 0, "scale factors need a source and a destination");
    DGB_REQUIRE(x_sf == nullptr || (sf_per_row >= 1 && x_sf_row_stride >= sf_per_row && rows_sf_row_stride >= sf_per_row && aligned_to(x_sf, 4) &&
                                    aligned_to(rows_sf, 4)),
                "scale rows must be 4-byte aligned and covered by their strides");
    PermuteParams p{};
    auto low = [](const void* q) { return static_cast<long long>(reinterpret_cast<uintptr_t>(q) & 15); };
    const int vec = vec_bytes_for({x_row_bytes, x_row_stride_bytes, rows_row_stride_bytes, low(x), low(rows)});
    p.rows.from = static_cast<const unsigned char*>(x);
    p.rows.to = static_cast<unsigned char*>(rows);
    p.rows.from_stride = x_row_stride_bytes;
    p.rows.to_stride = rows_row_stride_bytes;
    const int vec_used = vec == 16 || vec == 4 ? vec : (vec == 8 ? 4 : (vec == 2 ? 2 : 1));
    p.rows.row_vecs = x_row_bytes / vec_used;
    if (x_sf != nullptr && rows_sf != nullptr) {
        p.scales.from = reinterpret_cast<const unsigned char*>(x_sf);
        p.scales.to = reinterpret_cast<unsigned char*>(rows_sf);
        p.scales.from_stride = x_sf_row_stride * 4;
        p.scales.to_stride = rows_sf_row_stride * 4;
        p.scales.row_vecs = sf_per_row;
    }
    p.dest_row = dest_row;
    p.expert_end = expert_end;
    p.tokens = num_tokens;
    p.topk = num_topk;
    p.experts = num_experts;
    p.alignment = alignment;
    p.capacity = capacity;
    p.padding_blocks = zero_padding ? (alignment - 1 + 7) / 8 : 0;
    if ((num_tokens == 0 && p.padding_blocks == 0) || capacity == 0) return 0;
    int sms = 0;
    if (const int rc = effective_num_sms(&sms)) return rc;
    p.column_blocks = column_blocks(num_tokens, p.rows.row_vecs, 256, sms);
    const long long ctas = static_cast<long long>(num_tokens) * p.column_blocks + static_cast<long long>(num_experts) * p.padding_blocks;
    DGB_REQUIRE(ctas < (1ll << 31), "too many rows");
    const dim3 grid(static_cast<unsigned>(ctas));
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    switch (vec_used) {
        case 16: return launch_permute<uint4, uint32_t>(p, grid, stream);
        case 4: return launch_permute<uint32_t, uint32_t>(p, grid, stream);
        case 2: return launch_permute<unsigned short, uint32_t>(p, grid, stream);
        default: return launch_permute<unsigned char, uint32_t>(p, grid, stream);
    }
}

int dgb200_moe_unpermute(const void* rows, int64_t rows_row_stride, const float* topk_weights, const int32_t* dest_row, void* y, int64_t y_row_stride,
                         int32_t num_tokens, int32_t num_topk, int32_t hidden, int32_t capacity, int32_t is_fp32, void* stream) {
    UnpermuteParams p{};
    p.rows = rows;
    p.out = y;
    p.weights = topk_weights;
    p.dest_row = dest_row;
    p.rows_stride = rows_row_stride;
    p.out_stride = y_row_stride;
    p.tokens = num_tokens;
    p.topk = num_topk;
    p.hidden = hidden;
    p.experts = 1;
    p.alignment = 1;
    p.capacity = capacity;
    DGB_REQUIRE(num_tokens >= 0, "num_tokens must be >= 0");
    if (num_tokens == 0) return 0;
    return run_unpermute(p, false, is_fp32, static_cast<cudaStream_t>(stream));
}

int dgb200_moe_unpermute_backward(const void* dy, int64_t dy_row_stride, const void* rows, int64_t rows_row_stride, const float* topk_weights,
                                  const int32_t* dest_row, const int32_t* expert_end, void* d_rows, int64_t d_rows_row_stride, float* d_weights,
                                  int32_t num_tokens, int32_t num_topk, int32_t num_experts, int32_t alignment, int32_t hidden, int32_t capacity,
                                  int32_t is_fp32, void* stream) {
    UnpermuteParams p{};
    p.rows = rows;
    p.dy = dy;
    p.out = d_rows;
    p.d_weights = d_weights;
    p.weights = topk_weights;
    p.dest_row = dest_row;
    p.expert_end = expert_end;
    p.rows_stride = rows_row_stride;
    p.dy_stride = dy_row_stride;
    p.out_stride = d_rows_row_stride;
    p.tokens = num_tokens;
    p.topk = num_topk;
    p.hidden = hidden;
    p.experts = num_experts;
    p.alignment = alignment;
    p.capacity = capacity;
    return run_unpermute(p, true, is_fp32, static_cast<cudaStream_t>(stream));
}

int dgb200_swiglu(const void* x, int64_t x_row_stride, void* y, int64_t y_row_stride, int32_t rows, int32_t inter, const int32_t* grouped_layout,
                  int32_t num_groups, int32_t alignment, float activation_clamp, void* stream) {
    SwigluParams p{};
    p.x = static_cast<const __nv_bfloat16*>(x);
    p.out = y;
    p.x_stride = x_row_stride;
    p.out_stride = y_row_stride;
    p.layout = grouped_layout;
    p.num_groups = num_groups;
    p.alignment = alignment;
    p.rows = rows;
    p.inter = inter;
    p.clamp = activation_clamp;
    return run_swiglu(p, false, static_cast<cudaStream_t>(stream));
}

int dgb200_swiglu_backward(const void* dy, int64_t dy_row_stride, const void* x, int64_t x_row_stride, void* dx, int64_t dx_row_stride, int32_t rows,
                           int32_t inter, const int32_t* grouped_layout, int32_t num_groups, int32_t alignment, float activation_clamp, void* stream) {
    SwigluParams p{};
    p.x = static_cast<const __nv_bfloat16*>(x);
    p.dy = static_cast<const __nv_bfloat16*>(dy);
    p.out = dx;
    p.x_stride = x_row_stride;
    p.dy_stride = dy_row_stride;
    p.out_stride = dx_row_stride;
    p.layout = grouped_layout;
    p.num_groups = num_groups;
    p.alignment = alignment;
    p.rows = rows;
    p.inter = inter;
    p.clamp = activation_clamp;
    return run_swiglu(p, true, static_cast<cudaStream_t>(stream));
}

int dgb200_swiglu_per_token_cast_to_fp8(const void* x, int64_t x_row_stride, void* q, int64_t q_row_stride, float* sf, int64_t sf_row_stride,
                                        int32_t rows, int32_t inter, const int32_t* grouped_layout, int32_t num_groups, int32_t alignment,
                                        float activation_clamp, void* stream) {
    SwigluParams p{};
    p.x = static_cast<const __nv_bfloat16*>(x);
    p.out = q;
    p.sf = sf;
    p.x_stride = x_row_stride;
    p.out_stride = q_row_stride;
    p.sf_stride = sf_row_stride;
    p.layout = grouped_layout;
    p.num_groups = num_groups;
    p.alignment = alignment;
    p.rows = rows;
    p.inter = inter;
    p.clamp = activation_clamp;
    if (const int rc = check_swiglu(p, false, inter, 1)) return rc;
    DGB_REQUIRE(inter % 8 == 0 && x_row_stride % 8 == 0 && q_row_stride % 8 == 0 && aligned_to(x, 16) && aligned_to(q, 8),
                "inter must be a multiple of 8, rows of x 16-byte and of q 8-byte aligned");
    DGB_REQUIRE((sf != nullptr || rows == 0) && aligned_to(sf, 4) && sf_row_stride >= (inter + 127) / 128, "scale rows must hold one scale per 128 values");
    if (rows == 0) return 0;
    dim3 grid, block;
    int sms = 0;
    if (const int rc = effective_num_sms(&sms)) return rc;
    const bool many = swiglu_launch_shape(rows, (inter + 127) / 128 * 16, sms, &grid, &block) == kSwigluRows;
    DGB_REQUIRE(grid.y <= 65535u, "inter (%d) is too large", inter);
    DGB_CUDA(launch_kernel(many ? dgb200_swiglu_cast_kernel<kSwigluRows> : dgb200_swiglu_cast_kernel<1>, grid, block, 0, static_cast<cudaStream_t>(stream), use_pdl(), p));
    return 0;
}

}  // extern "C"
