/*
 * sample_accept.cpp -- the C ABI of the sampled accept: argument checks, work split and launches of
 * sample_accept.hip.
 */
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>

#include "verify_ops.h"

#ifndef DFQ_ACCEPT_HSACO_PATH
#error "DFQ_ACCEPT_HSACO_PATH must name the gfx950 code object to embed"
#endif
DFQ_EMBED(dfq_accept_hsaco, DFQ_ACCEPT_HSACO_PATH)

using namespace dfq;

namespace {

struct AcceptOps : LoadedOps {
    static constexpr OpsGroup kGroup = kAcceptOps;
    hipModule_t module = nullptr;
    hipFunction_t kernels[2][3] = {};   // [sums/weigh][bf16/f16/f32]
    dfq_status resolve() {
        static const char* kDt[3] = {"bf16", "f16", "f32"};
        hipError_t e = hipModuleLoadData(&module, dfq_accept_hsaco);
        if (e != hipSuccess) return hip_error(e, "hipModuleLoadData(gfx950 sampled-accept object)");
        char name[80];
        for (int k = 0; k < 2; ++k)
            for (int t = 0; t < 3; ++t) {
                snprintf(name, sizeof name, "dfq_accept_%s_%s", k ? "weigh" : "sums", kDt[t]);
                if ((e = hipModuleGetFunction(&kernels[k][t], module, name)) != hipSuccess)
                    return hip_error(e, name);
            }
        return DFQ_OK;
    }
    ~AcceptOps() override {
        if (module) (void)hipModuleUnload(module);
    }
};

dfq_status check_sizes(int batch, int rows, int V, dfq_dtype dtype) {
    if (batch < 1 || rows < 1 || V < 1)
        return fail(DFQ_ERR_INVALID_ARGUMENT, "batch, rows and V must be >= 1");
    if (rows > DFQ_ACCEPT_ROWS)
        return fail(DFQ_ERR_UNSUPPORTED, "at most %d rows (got %d)", DFQ_ACCEPT_ROWS, rows);
    if (batch > kMostGroups) return fail(DFQ_ERR_UNSUPPORTED, "too many sequences");
    if (V > 0x7fffffff / 2) return fail(DFQ_ERR_UNSUPPORTED, "V too large");
    if (dtype != DFQ_BF16 && dtype != DFQ_F16 && dtype != DFQ_F32)
        return fail(DFQ_ERR_UNSUPPORTED, "logits are bf16, fp16 or fp32");
    return DFQ_OK;
}

struct AcceptPlan {
    int all_rows, ranges, units, sums_apart, chunks;
    size_t sums, totals, arrived, bytes;   /* offsets; the parts come first */
};

constexpr int kWaves = DFQ_KV_THREADS / 64;

AcceptPlan plan_accept(int cus, int batch, int rows, int V, dfq_dtype dtype, bool drafted) {
    AcceptPlan a;
    a.all_rows = drafted ? 2 * rows - 1 : rows;
    const int unit = 64 * (dtype == DFQ_F32 ? 4 : 8);
    a.units = (V + unit - 1) / unit;
    a.sums_apart = drafted ? 6 * a.units : a.units;
    const int range = unit * DFQ_ACCEPT_PIECES;
    a.ranges = (V + range - 1) / range;
    /* Workgroups of a sequence: as many units a wave as leave no more than four workgroups a CU,
     * which are there at once (117 registers), and as few workgroups as that many units take: each
     * decides its sequence's drafts first.  With five a CU 64 sequences of seven drafts of 151936
     * tokens took 73.6 us for 71.9 and 16 32.3 for 29.9; eight took 33 rows of 50257 from 14.3 to
     * 16.2. */
    const auto parts = [](int n, int of) { return (int)(((int64_t)n + of - 1) / of); };
    const int most = std::max(1, 4 * cus / batch);
    a.chunks = parts(a.units, kWaves * parts(a.units, kWaves * most));
    const auto up = [](size_t n) { return (n + 255) & ~(size_t)255; };
    a.sums = up((size_t)batch * a.all_rows * a.ranges * sizeof(AcceptPart));
    a.totals = a.sums + up((size_t)batch * a.sums_apart * 8);
    a.arrived = a.totals + (drafted ? up((size_t)batch * a.chunks * 16) : 0);
    a.bytes = a.arrived + (size_t)batch * DFQ_ACCEPT_APART * 4;
    return a;
}

}  // namespace

extern "C" {

dfq_status dfq_sample_accept_workspace_bytes(dfq_ctx* ctx, int batch, int rows, int V,
                                             dfq_dtype dtype, int drafted, size_t* bytes) {
    if (!bytes) return fail(DFQ_ERR_INVALID_ARGUMENT, "null bytes");
    *bytes = 0;
    if (!ctx) return fail(DFQ_ERR_INVALID_ARGUMENT, "null context");
    const dfq_status s = check_sizes(batch, rows, V, dtype);
    if (s) return s;
    *bytes = plan_accept(dfq_num_cus(ctx), batch, rows, V, dtype, drafted && rows > 1).bytes;
    return DFQ_OK;
}

dfq_status dfq_sample_accept(dfq_ctx* ctx, const void* logits, int64_t batch_stride,
                             int64_t row_stride, const void* draft_logits,
                             int64_t draft_batch_stride, int64_t draft_row_stride, int batch,
                             int rows, int V, dfq_dtype dtype, const int32_t* drafts,
                             const int32_t* draft_lengths, const float* uniforms,
                             const float* temperatures, float temperature,
                             const float* draft_temperatures, float draft_temperature,
                             int32_t* tokens, int32_t* accepted, float* chances, void* workspace,
                             size_t workspace_bytes, void* stream) {
    if (!ctx) return fail(DFQ_ERR_INVALID_ARGUMENT, "null context");
    dfq_status s = check_sizes(batch, rows, V, dtype);
    if (s) return s;
    if (!logits || !uniforms || !tokens || !accepted)
        return fail(DFQ_ERR_INVALID_ARGUMENT, "null logits, uniforms, tokens or accepted");
    if (rows > 1 && !drafts) return fail(DFQ_ERR_INVALID_ARGUMENT, "null drafts");
    const bool drafted = draft_logits && rows > 1;
    if (batch_stride < 0 || row_stride < 0 ||
        (drafted && (draft_batch_stride < 0 || draft_row_stride < 0)))
        return fail(DFQ_ERR_INVALID_ARGUMENT, "negative stride");
    const size_t size = dtype_size(dtype);
    if (!aligned(logits, size) || !aligned(draft_logits, size) || !aligned(drafts, 4) ||
        !aligned(draft_lengths, 4) || !aligned(uniforms, 4) || !aligned(temperatures, 4) ||
        !aligned(draft_temperatures, 4) || !aligned(tokens, 4) || !aligned(accepted, 4) ||
        !aligned(chances, 4))
        return fail(DFQ_ERR_INVALID_ARGUMENT, "misaligned buffer");
    if ((!temperatures && !(temperature >= 0.0f && std::isfinite(temperature))) ||
        (drafted && !draft_temperatures &&
         !(draft_temperature >= 0.0f && std::isfinite(draft_temperature))))
        return fail(DFQ_ERR_INVALID_ARGUMENT, "temperatures are finite and not negative");
    const AcceptPlan a = plan_accept(dfq_num_cus(ctx), batch, rows, V, dtype, drafted);
    const int64_t jobs = (int64_t)batch * a.all_rows * a.ranges, groups = (jobs + kWaves - 1) / kWaves;
    const int64_t chunks = (int64_t)batch * a.chunks;
    if (groups > kMostGroups || chunks > kMostGroups)
        return fail(DFQ_ERR_UNSUPPORTED, "grid too large");
    if (!workspace || workspace_bytes < a.bytes)
        return fail(DFQ_ERR_WORKSPACE, "workspace of %zu bytes needed (got %zu)", a.bytes,
                    workspace ? workspace_bytes : (size_t)0);
    if (!aligned(workspace, 16))
        return fail(DFQ_ERR_INVALID_ARGUMENT, "workspace must be 16-byte aligned");
    char* const ws = (char*)workspace;
    AcceptParams p{};
    p.logits = logits;
    p.draft_logits = drafted ? draft_logits : nullptr;
    p.drafts = drafts;
    p.lengths = draft_lengths;
    p.uniforms = uniforms;
    p.temperatures = temperatures;
    p.draft_temperatures = draft_temperatures;
    p.tokens = tokens;
    p.accepted = accepted;
    p.chances = chances;
    p.parts = (AcceptPart*)ws;
    p.sums = (uint64_t*)(ws + a.sums);
    p.totals = (uint64_t*)(ws + a.totals);
    p.arrived = (int32_t*)(ws + a.arrived);
    p.batch_stride = batch_stride;
    p.row_stride = row_stride;
    p.draft_batch_stride = draft_batch_stride;
    p.draft_row_stride = draft_row_stride;
    int bits = 0;
    while ((V - 1) >> bits) ++bits;
    p.near = (drafted ? 2 : 1) * (1.75 * bits + 21.0) * 0x1p-24;   /* sample_accept.hip's bound */
    p.temperature = temperature;
    p.draft_temperature = draft_temperature;
    p.rows = rows;
    p.vocab = V;
    p.jobs = (int)jobs;
    p.units = a.units;
    p.sums_apart = a.sums_apart;
    p.all_rows = divisor(a.all_rows);
    p.ranges = divisor(a.ranges);
    p.chunks = divisor(a.chunks);
    const AcceptOps* ops;
    if ((s = ops_of(ctx, &ops))) return s;
    DeviceScope scope(ctx);
    void* args[] = {&p};
    hipError_t e = hipModuleLaunchKernel(ops->kernels[0][(int)dtype], (unsigned)groups, 1, 1,
                                         DFQ_KV_THREADS, 1, 1, 0, (hipStream_t)stream, args, nullptr);
    if (e == hipSuccess)
        e = hipModuleLaunchKernel(ops->kernels[1][(int)dtype], (unsigned)chunks, 1, 1,
                                  DFQ_KV_THREADS, 1, 1, 0, (hipStream_t)stream, args, nullptr);
    return e == hipSuccess ? DFQ_OK : hip_error(e, "launch dfq_sample_accept");
}

}  // extern "C"
