// tinym_grouped_host.inl -- launcher of the grouped and MXFP4 operators
// (tinym_grouped.cuh, tinym_mxfp4.cuh).  Part of tinym_capi.cu: it shares that
// file's error reporting and per-device state, and the kernels' device error
// word.

namespace {

using tinym::GroupedParams;
using tinym::MxParams;

// Tensor map of a stack of row-major uint8 matrices [experts, rows, cols].
// chunks == 1: {cols, rows, experts} in boxes of [box_rows x 128 bytes].
// chunks > 1: {128, rows, cols / 128, experts}, a box is `chunks` consecutive
// [box_rows x 128 bytes] tiles (a partial last chunk is left out).
// segs > 1: {128, rows, segs, cols / 128 / segs, experts}, each of the box's
// tiles has box_rows rows of every segment, one segment after the other.
// x: the X matrix, without the experts' dimension where that saves one.
// Past the end of any dimension a box reads zeros.
int encode_stack(const void* ptr, int64_t experts, int64_t rows, int64_t cols, int box_rows,
                 int chunks, int segs, bool x, CUtensorMap* out) {
    auto encode = get_encode();
    if (!encode)
        return fail(TINYM_ERR_CUDA, "cuTensorMapEncodeTiled unavailable (%s)",
                    cudaGetErrorString(g_encode_err));
    cuuint64_t dims[5], strides[4];
    cuuint32_t box[5], estr[5] = {1, 1, 1, 1, 1};
    int rank = 2;
    auto dim = [&](int64_t size, int64_t stride, int b) {
        dims[rank] = static_cast<cuuint64_t>(size);
        strides[rank - 1] = static_cast<cuuint64_t>(stride);
        box[rank++] = static_cast<cuuint32_t>(b);
    };
    dims[0] = static_cast<cuuint64_t>(chunks > 1 ? kBlockK : cols);
    box[0] = kBlockK;
    dims[1] = static_cast<cuuint64_t>(rows);
    box[1] = static_cast<cuuint32_t>(box_rows);
    strides[0] = static_cast<cuuint64_t>(cols);
    if (segs > 1) dim(segs, cols / segs, segs);
    if (chunks > 1) dim(cols / kBlockK / segs, kBlockK, chunks);
    if (!(x && segs > 1)) dim(experts, rows * cols, 1);
    const CUresult r = encode(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, rank, const_cast<void*>(ptr), dims,
                              strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, TINYM_L2_PROMOTION,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return fail(TINYM_ERR_CUDA,
                    "cuTensorMapEncodeTiled failed (CUresult %d) for [%lld x %lld x %lld]",
                    static_cast<int>(r), static_cast<long long>(experts),
                    static_cast<long long>(rows), static_cast<long long>(cols));
    return TINYM_OK;
}

int check_grouped(const void* x, const void* w, const void* y, int64_t ldy, int64_t rows,
                  int64_t experts, int64_t n, int64_t k, int k_step, const void* offsets,
                  const void* alpha, int32_t alpha_count, uint32_t flags) {
    if (!x || !w || !y) return fail(TINYM_ERR_INVALID_ARGUMENT, "X, W and Y must be non-null");
    if (rows < 1 || experts < 1 || n < 1 || k < 1)
        return fail(TINYM_ERR_INVALID_ARGUMENT,
                    "rows, experts, N and K must be positive (got %lld, %lld, %lld, %lld)",
                    (long long)rows, (long long)experts, (long long)n, (long long)k);
    if (k % k_step != 0)
        return fail(TINYM_ERR_UNSUPPORTED_SHAPE, "unsupported K=%lld: K must be a multiple of %d",
                    (long long)k, k_step);
    if (experts > tinym::kGrpMaxExperts)
        return fail(TINYM_ERR_UNSUPPORTED_SHAPE, "experts %lld > %d", (long long)experts,
                    tinym::kGrpMaxExperts);
    const int64_t lim = (int64_t(1) << 31) - 1024;
    if (rows > lim || n > lim || k > lim)
        return fail(TINYM_ERR_UNSUPPORTED_SHAPE, "rows, N or K exceeds the 32-bit index range");
    if (!offsets && experts != 1)
        return fail(TINYM_ERR_INVALID_ARGUMENT, "offsets may be NULL for one expert only");
    if (ldy < n) return fail(TINYM_ERR_INVALID_ARGUMENT, "ldy (%lld) < N (%lld)", (long long)ldy, (long long)n);
    if ((reinterpret_cast<uintptr_t>(x) & 15u) || (reinterpret_cast<uintptr_t>(w) & 15u))
        return fail(TINYM_ERR_MISALIGNED, "X and W must be 16-byte aligned");
    if (reinterpret_cast<uintptr_t>(y) & 1u) return fail(TINYM_ERR_MISALIGNED, "Y must be 2-byte aligned");
    if ((reinterpret_cast<uintptr_t>(offsets) & 3u) || (reinterpret_cast<uintptr_t>(alpha) & 3u))
        return fail(TINYM_ERR_MISALIGNED, "offsets and alpha must be 4-byte aligned");
    if (alpha && alpha_count != 1 && alpha_count != experts)
        return fail(TINYM_ERR_INVALID_ARGUMENT, "alpha has %d values, 1 or %lld are wanted", alpha_count,
                    (long long)experts);
    if (flags & ~static_cast<uint32_t>(TINYM_FLAG_ZERO_REST))
        return fail(TINYM_ERR_INVALID_ARGUMENT, "unknown flags 0x%x", flags);
    return TINYM_OK;
}

std::atomic<uint32_t> g_grouped_attr[kMaxDevices];
std::atomic<int> g_grouped_pairs[kMaxDevices];  // CTA pairs that are resident at once (0: not asked yet)

// Grid and attributes of a grouped launch; attrs holds 2 entries.
void grouped_config(const tinym::GroupedPlan& g, void* stream, cudaLaunchConfig_t* cfg,
                    cudaLaunchAttribute* attrs) {
    *cfg = cudaLaunchConfig_t{};
    cfg->gridDim = dim3(static_cast<unsigned>(g.grid));
    cfg->blockDim = dim3(tinym::kGrpThreads);
    cfg->dynamicSmemBytes = g.smem;
    cfg->stream = static_cast<cudaStream_t>(stream);
    attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[0].val.programmaticStreamSerializationAllowed = kUsePdl ? 1 : 0;
    attrs[1].id = cudaLaunchAttributeClusterDimension;
    attrs[1].val.clusterDim.x = 2;
    attrs[1].val.clusterDim.y = 1;
    attrs[1].val.clusterDim.z = 1;
    cfg->attrs = attrs;
    cfg->numAttrs = g.pair ? 2 : 1;
}

// k_bytes: bytes of one operand row.  x_scales / w_scales: MXFP4, else null.
int grouped_impl(bool fp4, const void* x, const void* x_scales, const void* w, const void* w_scales,
                 void* y, int64_t ldy, int64_t rows, int64_t experts, int64_t n, int64_t k_bytes,
                 const int32_t* offsets, const float* alpha, int32_t alpha_count, uint32_t flags,
                 void* stream, uint64_t timeout_ns = kDefaultTimeoutNs, uint32_t selftest = 0u) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
    DeviceInfo* di = nullptr;
    int st = device_info(dev, &di);
    if (st != TINYM_OK) return st;
    tinym::GroupedPlan g;
    if (const char* why = tinym::grouped_plan(fp4, rows, experts, n, k_bytes, di->sm_count, kSmemLimit, &g))
        return fail(TINYM_ERR_UNSUPPORTED_SHAPE, "%s (rows %lld, experts %lld, N %lld)", why,
                    (long long)rows, (long long)experts, (long long)n);
    GroupedParams& p = g.prm;
    // A map per box height that the pieces can have.
    const int segs = std::max(1, p.fold);
    const int chunks = g.pair || k_bytes < kBlockK ? 1 : tinym::grouped_chunks(g.mode);
    const bool tail = !g.pair && !p.chunked;
    tinym::GroupedMaps maps;
    for (int i = g.pair ? tinym::kBlockUnits - 1 : 0; i < p.piece_units; ++i) {
        if ((st = encode_stack(w, experts, n, k_bytes, 8 * (i + 1), chunks, segs, false, &maps.w[i])) !=
            TINYM_OK)
            return st;
        if (tail && (st = encode_stack(w, experts, n, k_bytes, 8 * (i + 1), 1, 1, false,
                                       &maps.w_tail[i])) != TINYM_OK)
            return st;
    }
    const int64_t x_most = p.fold ? p.fold_x : std::min<int64_t>(p.tn, rows);
    for (int i = 0; i < 4; ++i) {
        const int box = tinym::grouped_x_box(g.pair, i);
        if ((st = encode_stack(x, 1, rows, k_bytes, box, chunks, segs, true, &maps.x[i])) != TINYM_OK)
            return st;
        if (tail && (st = encode_stack(x, 1, rows, k_bytes, box, 1, 1, true, &maps.x_tail[i])) != TINYM_OK)
            return st;
        if (box * (g.pair ? 2 : 1) >= x_most) break;
    }
    p.y = static_cast<__nv_bfloat16*>(y);
    p.ldy = ldy;
    p.wide_y = ldy % 8 == 0 && (reinterpret_cast<uintptr_t>(y) & 15u) == 0;
    p.offsets = offsets;
    p.alpha = alpha;
    p.alpha_stride = alpha_count > 1 ? 1 : 0;
    p.x_scales = static_cast<const uint8_t*>(x_scales);
    p.w_scales = static_cast<const uint8_t*>(w_scales);
    if (fp4)
        p.w_scale_stride = (n + 127) / 128 * ((2 * k_bytes + 127) / 128) * tinym::kScaleBlock;
    p.flags = (flags & TINYM_FLAG_ZERO_REST ? tinym::kGrpZeroRest : 0u) | selftest;
    p.timeout_ns = timeout_ns;
    if ((st = pending_word(di, true, &p.err_host)) != TINYM_OK) return st;

#define TINYM_GROUPED(F, M) reinterpret_cast<const void*>(&tinym::tinym_grouped_kernel<F, tinym::M>)
    static const void* const kFn[2][3] = {
        {TINYM_GROUPED(false, kStream), TINYM_GROUPED(false, kFold), TINYM_GROUPED(false, kPair)},
        {TINYM_GROUPED(true, kStream), TINYM_GROUPED(true, kFold), TINYM_GROUPED(true, kPair)}};
#undef TINYM_GROUPED
    const void* fn = kFn[fp4 ? 1 : 0][g.mode];
    const uint32_t bit = 1u << ((fp4 ? 3 : 0) + g.mode);
    if (!(g_grouped_attr[dev].load(std::memory_order_acquire) & bit)) {
        e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit);
        if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(MaxDynamicSharedMemorySize)");
        g_grouped_attr[dev].fetch_or(bit, std::memory_order_acq_rel);
    }
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attrs[2];
    grouped_config(g, stream, &cfg, attrs);
    if (g.pair) {
        // Pairs need two SMs of one cluster: a persistent grid of more pairs
        // than are resident at once would run its last ones alone.  One count
        // serves every call: a pair's CTAs always take all shared memory.
        int pairs = g_grouped_pairs[dev].load(std::memory_order_relaxed);
        if (!pairs) {
            e = cudaOccupancyMaxActiveClusters(&pairs, fn, &cfg);
            if (e != cudaSuccess) return cuda_fail(e, "cudaOccupancyMaxActiveClusters");
            if (pairs < 1) return fail(TINYM_ERR_CUDA, "no CTA pair fits the device");
            g_grouped_pairs[dev].store(pairs, std::memory_order_relaxed);
        }
        if (g.grid > 2 * pairs) cfg.gridDim.x = static_cast<unsigned>(2 * pairs);
    }
    void* args[2] = {&maps, &p};
    e = cudaLaunchKernelExC(&cfg, fn, args);
    if (e != cudaSuccess) return cuda_fail(e, "grouped kernel launch");
    return TINYM_OK;
}

int check_scales(const void* xs, const void* ws) {
    if (!xs || !ws) return fail(TINYM_ERR_INVALID_ARGUMENT, "X and W scales must be non-null");
    if ((reinterpret_cast<uintptr_t>(xs) & 15u) || (reinterpret_cast<uintptr_t>(ws) & 15u))
        return fail(TINYM_ERR_MISALIGNED, "scales must be 16-byte aligned");
    return TINYM_OK;
}

// run: columns that one warp takes (256 * kMxSteps).
int mx_params(int64_t batch, int64_t rows, int64_t k, int64_t run, MxParams* p) {
    if (batch < 1 || rows < 1 || k < 1)
        return fail(TINYM_ERR_INVALID_ARGUMENT, "batch, rows and K must be positive (got %lld, %lld, %lld)",
                    (long long)batch, (long long)rows, (long long)k);
    if (k % 32 != 0)
        return fail(TINYM_ERR_UNSUPPORTED_SHAPE, "unsupported K=%lld: K must be a multiple of 32",
                    (long long)k);
    const int64_t lim = int64_t(1) << 30;  // of the kernels' 32-bit indices
    const int64_t kc = (k + 127) / 128, rb = (rows + 127) / 128, pad = rb * 128 - rows;
    if (batch > lim || rows > lim || k > lim || batch * rows > lim || batch * rows > lim / kc ||
        (pad && batch > lim / (pad * kc)))
        return fail(TINYM_ERR_UNSUPPORTED_SHAPE, "batch * rows * K exceeds the 32-bit index range");
    p->rows = static_cast<int32_t>(rows);
    p->k = static_cast<int32_t>(k);
    p->row_blocks = static_cast<int32_t>(rb);
    const int64_t per_row = (k + run - 1) / run;
    p->runs = static_cast<uint32_t>(batch * rows * per_row);
    p->pad_words = static_cast<uint32_t>(batch * pad * kc);
    p->per_row = tinym::FastDiv::make(static_cast<uint32_t>(per_row));
    p->kc = tinym::FastDiv::make(static_cast<uint32_t>(kc));
    p->per_matrix = tinym::FastDiv::make(static_cast<uint32_t>(rows));
    p->pad_per_matrix = tinym::FastDiv::make(static_cast<uint32_t>(std::max<int64_t>(1, pad)));
    return TINYM_OK;
}

int mx_launch(bool quantize, const void* wide, int32_t dtype, const void* codes, const void* scales,
              int64_t batch, int64_t rows, int64_t k, void* stream) {
    if (!wide || !codes || !scales)
        return fail(TINYM_ERR_INVALID_ARGUMENT, "values, codes and scales must be non-null");
    if (dtype != TINYM_ACT_BF16 && dtype != TINYM_ACT_F32)
        return fail(TINYM_ERR_INVALID_ARGUMENT, "dtype %d is not TINYM_ACT_BF16 / TINYM_ACT_F32", dtype);
    MxParams p{};
    const int64_t run = 256 * (dtype == TINYM_ACT_BF16 ? tinym::kMxSteps<__nv_bfloat16> : tinym::kMxSteps<float>);
    int st = mx_params(batch, rows, k, run, &p);
    if (st != TINYM_OK) return st;
    if ((reinterpret_cast<uintptr_t>(wide) & 15u) || (reinterpret_cast<uintptr_t>(codes) & 15u) ||
        (reinterpret_cast<uintptr_t>(scales) & 15u))
        return fail(TINYM_ERR_MISALIGNED, "values, codes and scales must be 16-byte aligned");
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
    DeviceInfo* di = nullptr;
    if ((st = device_info(dev, &di)) != TINYM_OK) return st;
    constexpr int kWarps = tinym::kMxThreads / 32;
    const int64_t want = std::max<int64_t>(
        (p.runs + kWarps - 1) / kWarps,
        quantize ? (p.pad_words + tinym::kMxThreads - 1) / tinym::kMxThreads : 1);
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>(want, int64_t(di->sm_count) * 8));
    static const void* const kFn[2][2] = {
        {reinterpret_cast<const void*>(&tinym::tinym_mxfp4_dequantize_kernel<float>),
         reinterpret_cast<const void*>(&tinym::tinym_mxfp4_dequantize_kernel<__nv_bfloat16>)},
        {reinterpret_cast<const void*>(&tinym::tinym_mxfp4_quantize_kernel<float>),
         reinterpret_cast<const void*>(&tinym::tinym_mxfp4_quantize_kernel<__nv_bfloat16>)}};
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(tinym::kMxThreads);
    cfg.stream = static_cast<cudaStream_t>(stream);
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = kUsePdl ? 1 : 0;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    // quantise: x, codes, scales; dequantise: codes, scales, y
    void* q_args[4] = {&wide, &codes, &scales, &p};
    void* d_args[4] = {&codes, &scales, &wide, &p};
    e = cudaLaunchKernelExC(&cfg, kFn[quantize ? 1 : 0][dtype == TINYM_ACT_BF16 ? 1 : 0],
                            quantize ? q_args : d_args);
    if (e != cudaSuccess) return cuda_fail(e, "MXFP4 kernel launch");
    return TINYM_OK;
}

}  // namespace

extern "C" {

int tinym_fp8_gemm_grouped(const void* x, const void* w, void* y, int64_t ldy, int64_t rows,
                           int64_t experts, int64_t n, int64_t k, const int32_t* offsets_dev,
                           const float* alpha_dev, int32_t alpha_count, uint32_t flags,
                           void* stream) {
    t_last_error[0] = '\0';
    const int st = check_grouped(x, w, y, ldy, rows, experts, n, k, 16, offsets_dev, alpha_dev,
                                 alpha_count, flags);
    if (st != TINYM_OK) return st;
    return grouped_impl(false, x, nullptr, w, nullptr, y, ldy, rows, experts, n, k, offsets_dev,
                        alpha_dev, alpha_count, flags, stream);
}

int tinym_selftest_grouped_timeout(const void* x, const void* w, void* y, int64_t rows,
                                   int64_t experts, int64_t n, int64_t k, const int32_t* offsets_dev,
                                   uint64_t timeout_ns, void* stream) {
    t_last_error[0] = '\0';
    if (timeout_ns == 0 || timeout_ns > 10ull * kDefaultTimeoutNs)
        return fail(TINYM_ERR_INVALID_ARGUMENT, "timeout_ns must be in 1 .. 1e10");
    const int st = check_grouped(x, w, y, n, rows, experts, n, k, 16, offsets_dev, nullptr, 0, 0u);
    if (st != TINYM_OK) return st;
    return grouped_impl(false, x, nullptr, w, nullptr, y, n, rows, experts, n, k, offsets_dev, nullptr,
                        0, 0u, stream, timeout_ns, tinym::kGrpNoLoads);
}

int tinym_selftest_grouped_lost(int32_t lost, const void* x, const void* x_scales, const void* w,
                                const void* w_scales, void* y, int64_t rows, int64_t experts,
                                int64_t n, int64_t k, const int32_t* offsets_dev,
                                uint64_t timeout_ns, void* stream) {
    t_last_error[0] = '\0';
    static const uint32_t kLost[3] = {tinym::kGrpNoLoads, tinym::kGrpNoMma, tinym::kGrpNoCommit};
    if (lost < 0 || lost > 2) return fail(TINYM_ERR_INVALID_ARGUMENT, "lost must be 0, 1 or 2 (got %d)", lost);
    if (timeout_ns == 0 || timeout_ns > 10ull * kDefaultTimeoutNs)
        return fail(TINYM_ERR_INVALID_ARGUMENT, "timeout_ns must be in 1 .. 1e10");
    const bool fp4 = x_scales || w_scales;
    int st = check_grouped(x, w, y, n, rows, experts, n, k, fp4 ? 32 : 16, offsets_dev, nullptr, 0, 0u);
    if (st == TINYM_OK && fp4) st = check_scales(x_scales, w_scales);
    if (st != TINYM_OK) return st;
    return grouped_impl(fp4, x, x_scales, w, w_scales, y, n, rows, experts, n, fp4 ? k / 2 : k, offsets_dev,
                        nullptr, 0, 0u, stream, timeout_ns, kLost[lost]);
}

int tinym_mxfp4_gemm_grouped(const void* x, const void* x_scales, const void* w,
                             const void* w_scales, void* y, int64_t ldy, int64_t rows,
                             int64_t experts, int64_t n, int64_t k, const int32_t* offsets_dev,
                             const float* alpha_dev, int32_t alpha_count, uint32_t flags,
                             void* stream) {
    t_last_error[0] = '\0';
    int st = check_grouped(x, w, y, ldy, rows, experts, n, k, 32, offsets_dev, alpha_dev,
                           alpha_count, flags);
    if (st != TINYM_OK) return st;
    if ((st = check_scales(x_scales, w_scales)) != TINYM_OK) return st;
    return grouped_impl(true, x, x_scales, w, w_scales, y, ldy, rows, experts, n, k / 2, offsets_dev,
                        alpha_dev, alpha_count, flags, stream);
}

int tinym_mxfp4_gemm(const void* x, const void* x_scales, const void* w, const void* w_scales,
                     void* y, int64_t ldy, int64_t m, int64_t n, int64_t k, const float* alpha_dev,
                     void* stream) {
    return tinym_mxfp4_gemm_grouped(x, x_scales, w, w_scales, y, ldy, m, 1, n, k, nullptr, alpha_dev,
                                    1, 0u, stream);
}

int tinym_mxfp4_scale_bytes(int64_t batch, int64_t rows, int64_t k, int64_t* bytes) {
    t_last_error[0] = '\0';
    if (!bytes) return fail(TINYM_ERR_INVALID_ARGUMENT, "bytes is NULL");
    MxParams p{};
    const int st = mx_params(batch, rows, k, 128, &p);
    if (st != TINYM_OK) return st;
    *bytes = batch * p.row_blocks * p.kc.d * tinym::kScaleBlock;
    return TINYM_OK;
}

int tinym_mxfp4_quantize(const void* x, int32_t dtype, void* codes, void* scales, int64_t batch,
                         int64_t rows, int64_t k, void* stream) {
    t_last_error[0] = '\0';
    return mx_launch(true, x, dtype, codes, scales, batch, rows, k, stream);
}

int tinym_mxfp4_dequantize(const void* codes, const void* scales, void* y, int32_t dtype,
                           int64_t batch, int64_t rows, int64_t k, void* stream) {
    t_last_error[0] = '\0';
    return mx_launch(false, y, dtype, codes, scales, batch, rows, k, stream);
}

}  // extern "C"
