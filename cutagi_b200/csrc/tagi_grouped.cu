// Linear layers grouped by expert: rows [offsets[e], offsets[e + 1]) of the dispatch order go through expert e's weights.
// The offsets and the gather index are device data, so no pass waits for the host; both are checked where they are read
// (offsets are clamped to [0, S] and made non-decreasing, a row whose token lies outside [0, R) reads as zero).
#include "tagi_grouped.h"

namespace tagi {
namespace {

int run(int pass, GroupedArgs &a, cudaStream_t st) {
    a.few = pass == PARAM ? FEW_PARAM_ROWS : FEW_ROWS;
    int rc = grouped_few(pass, a, st);
    if (rc != TAGI_OK || a.S <= a.few) return rc;
    if (pass == FWD && (rc = grouped_second_moment(a, st)) != TAGI_OK) return rc;
    if (pass != PARAM && (rc = grouped_thin(pass, a, st)) != TAGI_OK) return rc;
    return pass != PARAM && a.S <= THIN_ROWS ? TAGI_OK : grouped_tc(pass, a, st);
}

bool sizes_fit(int E, int S, int K, int N) {
    return E >= 1 && E <= 1024 && S >= 0 && S <= (1 << 28) && K >= 1 && K <= (1 << 20) && N >= 1 && N <= (1 << 20);
}
// Workspace: partial sums of the tensor-core kernels, which use it one after the other, then, forward, mu_a^2 + var_a; nothing
// where the number of rows in all rules these kernels out.
size_t parts_bytes(int pass, int E, int S, int K, int N) {
    const size_t thin = pass == PARAM || S <= FEW_ROWS ? 0 : grouped_thin_parts_bytes(pass, E, S, K, N);
    const size_t tc = S <= (pass == PARAM ? FEW_PARAM_ROWS : THIN_ROWS) ? 0 : grouped_tc_parts_bytes(pass, E, S, K, N);
    return thin > tc ? thin : tc;
}
size_t second_bytes(int S, int R, int K) { return S <= FEW_ROWS ? 0 : (size_t)R * K * sizeof(float); }

int check_workspace(const char *who, int pass, const GroupedArgs &a, const void *workspace, size_t bytes) {
    const size_t need = tagi_grouped_linear_workspace_bytes(pass, a.E, a.S, a.R, a.K, a.N);
    if (need > 0 && (workspace == nullptr || !aligned16(workspace) || bytes < need))
        return fail(TAGI_ERR_INVALID_ARGUMENT,
                    std::string(who) + ": workspace is null, not 16-byte aligned or smaller than tagi_grouped_linear_workspace_bytes");
    return TAGI_OK;
}

int check_grouped(const char *who, int E, int S, int K, int N, const int *offsets) {
    if (sizes_fit(E, S, K, N) && offsets != nullptr && aligned4(offsets)) return TAGI_OK;
    if (E < 1 || E > 1024 || S < 0 || K < 1 || N < 1)
        return fail(TAGI_ERR_INVALID_ARGUMENT, std::string(who) + ": 1 to 1024 experts, positive feature counts, rows must not be negative");
    if (K > (1 << 20) || N > (1 << 20) || S > (1 << 28))
        return fail(TAGI_ERR_INVALID_ARGUMENT, std::string(who) + ": more than 2^20 features or 2^28 rows");
    return fail(TAGI_ERR_INVALID_ARGUMENT, std::string(who) + ": offsets is null or not 4-byte aligned");
}

}  // namespace
}  // namespace tagi

using namespace tagi;

#define TAGI_PTR(p) TAGI_REQUIRE((p) != nullptr && aligned4(p), #p " is null or not 4-byte aligned")

extern "C" {

size_t tagi_grouped_linear_workspace_bytes(int pass, int E, int S, int R, int K, int N) {
    if (pass < FWD || pass > PARAM || !sizes_fit(E, S, K, N) || R < 0) return 0;
    return parts_bytes(pass, E, S, K, N) + (pass == FWD ? second_bytes(S, R, K) : 0);
}

int tagi_grouped_linear_fwd(int E, int S, int R, int K, int N, int has_bias, const int *offsets, const int *token,
                            const float *mu_w, const float *var_w, const float *mu_b, const float *var_b, const float *mu_a,
                            const float *var_a, float *mu_z, float *var_z, void *workspace, size_t workspace_bytes, void *stream) {
    int rc = check_grouped(__func__, E, S, K, N, offsets);
    if (rc != TAGI_OK) return rc;
    TAGI_PTR(mu_w);
    TAGI_PTR(var_w);
    if (has_bias) {
        TAGI_PTR(mu_b);
        TAGI_PTR(var_b);
    }
    TAGI_REQUIRE(token == nullptr || aligned4(token), "token is not 4-byte aligned");
    TAGI_REQUIRE(R >= 0, "input rows must not be negative");
    if (S == 0) return TAGI_OK;
    TAGI_REQUIRE(token != nullptr || R == S, "without a gather index the input has as many rows as the output");
    TAGI_REQUIRE(R > 0, "rows to compute but no input rows");
    TAGI_PTR(mu_a);
    TAGI_PTR(var_a);
    TAGI_PTR(mu_z);
    TAGI_PTR(var_z);
    GroupedArgs a{};
    a.E = E, a.S = S, a.R = R, a.K = K, a.N = N, a.offsets = offsets, a.token = token, a.mu_w = mu_w, a.var_w = var_w;
    a.mu_b = has_bias ? mu_b : nullptr, a.var_b = has_bias ? var_b : nullptr, a.a0 = mu_a, a.a1 = var_a, a.o0 = mu_z, a.o1 = var_z;
    if ((rc = check_workspace(__func__, FWD, a, workspace, workspace_bytes)) != TAGI_OK) return rc;
    a.parts = static_cast<float *>(workspace);
    a.second = a.parts + parts_bytes(FWD, E, S, K, N) / sizeof(float);
    return run(FWD, a, static_cast<cudaStream_t>(stream));
}

int tagi_grouped_linear_bwd_state(int E, int S, int K, int N, const int *offsets, const float *mu_w, const float *jcb,
                                  const float *dmu_z, const float *dvar_z, float *dmu_a, float *dvar_a, void *workspace,
                                  size_t workspace_bytes, void *stream) {
    int rc = check_grouped(__func__, E, S, K, N, offsets);
    if (rc != TAGI_OK) return rc;
    TAGI_PTR(mu_w);
    TAGI_REQUIRE(jcb == nullptr || aligned4(jcb), "jcb is not 4-byte aligned");
    if (S == 0) return TAGI_OK;
    TAGI_PTR(dmu_z);
    TAGI_PTR(dvar_z);
    TAGI_PTR(dmu_a);
    TAGI_PTR(dvar_a);
    GroupedArgs a{};
    a.E = E, a.S = S, a.R = S, a.K = K, a.N = N, a.offsets = offsets, a.mu_w = mu_w, a.jcb = jcb, a.a0 = dmu_z, a.a1 = dvar_z;
    a.o0 = dmu_a, a.o1 = dvar_a;
    if ((rc = check_workspace(__func__, STATE, a, workspace, workspace_bytes)) != TAGI_OK) return rc;
    a.parts = static_cast<float *>(workspace);
    return run(STATE, a, static_cast<cudaStream_t>(stream));
}

int tagi_grouped_linear_bwd_param(int E, int S, int R, int K, int N, int has_bias, const int *offsets, const int *token,
                                  const float *var_w, const float *var_b, const float *mu_a, const float *dmu_z,
                                  const float *dvar_z, float *dmu_w, float *dvar_w, float *dmu_b, float *dvar_b, void *workspace,
                                  size_t workspace_bytes, void *stream) {
    int rc = check_grouped(__func__, E, S, K, N, offsets);
    if (rc != TAGI_OK) return rc;
    TAGI_PTR(var_w);
    TAGI_PTR(dmu_w);
    TAGI_PTR(dvar_w);
    if (has_bias) {
        TAGI_PTR(var_b);
        TAGI_PTR(dmu_b);
        TAGI_PTR(dvar_b);
    }
    TAGI_REQUIRE(token == nullptr || aligned4(token), "token is not 4-byte aligned");
    TAGI_REQUIRE(R >= 0, "input rows must not be negative");
    if (S > 0) {
        TAGI_REQUIRE(token != nullptr || R == S, "without a gather index the input has as many rows as the deltas");
        TAGI_REQUIRE(R > 0, "deltas but no input rows");
        TAGI_PTR(mu_a);
        TAGI_PTR(dmu_z);
        TAGI_PTR(dvar_z);
    }
    GroupedArgs a{};
    a.E = E, a.S = S, a.R = R, a.K = K, a.N = N, a.offsets = offsets, a.token = token, a.var_w = var_w, a.x = mu_a;
    a.var_b = has_bias ? var_b : nullptr, a.a0 = dmu_z, a.a1 = dvar_z, a.o0 = dmu_w, a.o1 = dvar_w, a.ob0 = dmu_b, a.ob1 = dvar_b;
    if ((rc = check_workspace(__func__, PARAM, a, workspace, workspace_bytes)) != TAGI_OK) return rc;
    a.parts = static_cast<float *>(workspace);
    return run(PARAM, a, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
