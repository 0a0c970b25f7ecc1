// Entry points of the 4-bit matrices: argument validation in the order of the other entries (ops.cpp), then one launch.
#include "op_common.h"
#include "q4.h"

using namespace t2sp;

namespace t2sp {
namespace {

int resolve_group(const t2sp_q4_desc* desc, int* group) {
    *group = desc && desc->group ? desc->group : 64;
    if (*group != 32 && *group != 64 && *group != 128) return constraint("q4.desc.group", *group, "32, 64 or 128", 64);
    return 0;
}

// Packed matrices and scales lie densely, as a bounds query describes them.
int check_packed(const Arg& a, const int* ext, int align) {
    int64_t stride = 1;
    for (int d = 0; d < 4; ++d) {
        const std::string v = std::string(a.name);
        if (a.b->dim[d].min != 0) return constraint((v + ".min." + std::to_string(d)).c_str(), a.b->dim[d].min, "0", 0);
        if (a.b->dim[d].extent != ext[d])
            return constraint((v + ".extent." + std::to_string(d)).c_str(), a.b->dim[d].extent, "the packed extent", ext[d]);
        if (ext[d] > 1 && a.b->dim[d].stride != stride)
            return constraint((v + ".stride." + std::to_string(d)).c_str(), a.b->dim[d].stride, "the dense stride",
                              static_cast<int>(std::min<int64_t>(stride, 0x7fffffff)));
        stride *= ext[d];
    }
    if (buf_on_our_device(a.b) && (a.b->device & uint64_t(align - 1)))
        return constraint((std::string(a.name) + ".device").c_str(), static_cast<int>(a.b->device & uint64_t(align - 1)), "a multiple of", align);
    return 0;
}

template <class Launch>
int run_q4(const char* who, Q4Params& p, bool sync_after, Launch launch) {
    cudaStream_t s = rt_stream();
    p.status = rt_status_word();
    p.wait_cycles = rt_env().wait_cycles;
    p.skip_stage = rt_env().test_skip_stage;
    if (sync_after) cudaEventRecord(rt_event(0), s);
    const cudaError_t e = launch(p, s);
    if (e != cudaSuccess) {
        fprintf(stderr, "t2sp_b200: %s: kernel launch failed: %s\n", who, cudaGetErrorString(e));
        return halide_error_code_device_run_failed;
    }
    rt_count_launch(1);
    if (sync_after) cudaEventRecord(rt_event(1), s);
    return 0;
}

// Extents of the packed form of an (N, K, E) matrix.
void packed_extents(int N, int K, int E, int group, int* q, int* s) {
    q[0] = 512; q[1] = q4_kblocks(K); q[2] = q4_strips(N); q[3] = E;
    s[0] = 16; s[1] = q4_groups(K, group); s[2] = q4_strips(N); s[3] = E;
}

// The K and N that a packed matrix holds at the most, within the limit of extents.
int packed_most(const Arg& q, int* K, int* N) {
    for (int d = 1; d < 3; ++d) {
        const int64_t most = int64_t(q.b->dim[d].extent) * (d == 1 ? 64 : 16);
        if (most > (1 << 30)) return halide_error_buffer_extents_too_large(nullptr, q.name, most, int64_t(1) << 30);
        *(d == 1 ? K : N) = static_cast<int>(most);
    }
    return 0;
}

// Bounds queries of q4_pack and q4_unpack: the packed shapes from W, or the largest W that the packed shapes hold.
int query_w_q_s(Arg* args, int w, int q, int s, int tb, int group) {
    halide_buffer_t *W = args[w].b, *Q = args[q].b, *S = args[s].b;
    if (int e = check_query_known(args, 3)) return e;
    if (buf_is_bounds_query(W)) {
        if (buf_is_bounds_query(Q)) return halide_error_host_is_null(nullptr, args[w].role().c_str());
        if (int e = check_type_dims(args[q], kU8)) return e;
        const uint32_t t = buf_is_bounds_query(S) ? kBF16 : buf_type_word(S);
        int N = 0, K = 0;
        if (int e = packed_most(args[q], &K, &N)) return e;
        const int we[3] = {tb ? K : N, tb ? N : K, Q->dim[3].extent};
        fill_query(W, t, 3, we);
    } else {
        const uint32_t t = buf_type_word(W);
        if (t != kBF16 && t != kF16) return halide_error_bad_type(nullptr, args[w].role().c_str(), t, kBF16);
        if (int e = check_type_dims(args[w], t)) return e;
    }
    int qe[4], se[4];
    packed_extents(W->dim[tb ? 1 : 0].extent, W->dim[tb ? 0 : 1].extent, W->dim[2].extent, group, qe, se);
    const uint32_t t = buf_type_word(W);
    if (buf_is_bounds_query(Q)) fill_query(Q, kU8, 4, qe);
    if (buf_is_bounds_query(S)) fill_query(S, t, 4, se);
    return 0;
}

// W with Q and S: the checks that q4_pack and q4_unpack share.
int check_w_q_s(Arg* args, int w, int q, int s, int tb, int group) {
    const uint32_t t = buf_type_word(args[w].b);
    if (t != kBF16 && t != kF16) return halide_error_bad_type(nullptr, args[w].role().c_str(), t, kBF16);
    if (int e = check_type_dims(args[w], t)) return e;
    if (int e = check_type_dims(args[q], kU8)) return e;
    if (int e = check_type_dims(args[s], t)) return e;
    for (int i = 0; i < 3; ++i)
        if (int e = check_extents_nonneg(args[i])) return e;
    if (int e = check_extent_limit(args[w])) return e;
    if (int e = check_min0(args[w])) return e;
    if (int e = check_stride0(args[w])) return e;
    if (int e = check_strides(args[w])) return e;
    for (int i = 0; i < 3; ++i)
        if (int e = check_sizes(args[i])) return e;
    if (int e = check_device_address(args[w])) return e;
    const halide_buffer_t* W = args[w].b;
    int qe[4], se[4];
    packed_extents(W->dim[tb ? 1 : 0].extent, W->dim[tb ? 0 : 1].extent, W->dim[2].extent, group, qe, se);
    if (int e = check_packed(args[q], qe, 16)) return e;
    if (int e = check_packed(args[s], se, 16)) return e;
    for (int i = 0; i < 3; ++i)
        if (int e = check_host(args[i])) return e;
    return 0;
}

}  // namespace
}  // namespace t2sp

extern "C" int t2sp_b200_q4_pack(halide_buffer_t* W, halide_buffer_t* Q, halide_buffer_t* S, const t2sp_q4_desc* desc) {
    Arg args[3] = {{W, "W", false, 3}, {Q, "Q", true, 4}, {S, "S", true, 4}};
    if (int e = check_null(args, 3)) return e;
    int group = 0;
    if (int e = resolve_group(desc, &group)) return e;
    const int tb = desc && desc->trans_b ? 1 : 0;
    if (buf_is_bounds_query(W) || buf_is_bounds_query(Q) || buf_is_bounds_query(S)) return query_w_q_s(args, 0, 1, 2, tb, group);
    if (int e = check_w_q_s(args, 0, 1, 2, tb, group)) return e;
    Q4Params p = {};
    p.N = W->dim[tb ? 1 : 0].extent; p.K = W->dim[tb ? 0 : 1].extent; p.E = W->dim[2].extent;
    if (p.N == 0 || p.K == 0 || p.E == 0) return 0;

    if (int e = rt_ensure_device()) return e;
    const bool sync_after = !(all_resident({W, Q, S}) && tls().async);
    if (int e = check_capture("q4_pack", sync_after, false)) return e;
    Views vw;
    if (int e = rt_input_view(W, "W", &vw.v[vw.n])) return e;
    vw.n++;
    for (int i = 1; i < 3; ++i, ++vw.n)
        if (int e = rt_output_view(args[i].b, args[i].name, &vw.v[vw.n])) return e;
    p.w = vw.v[0].ptr;
    p.w_end = static_cast<const uint16_t*>(p.w) + buf_elems_span(W);
    p.ldw = W->dim[1].stride; p.bs_w = W->dim[2].stride;
    p.trans_b = tb; p.group = group; p.bf16 = buf_type_word(W) == kBF16;
    p.q = static_cast<uint8_t*>(vw.v[1].ptr);
    p.s = static_cast<uint16_t*>(vw.v[2].ptr);
    if (int e = run_q4("q4_pack", p, sync_after, q4_pack_launch)) return e;
    for (int i = 1; i < 3; ++i)
        if (int e = rt_finish_output(args[i].b, args[i].name, &vw.v[i])) return e;
    return finish_call("q4_pack", "kernel_Out", sync_after);
}

extern "C" int t2sp_b200_q4_unpack(halide_buffer_t* Q, halide_buffer_t* S, halide_buffer_t* W, const t2sp_q4_desc* desc) {
    Arg args[3] = {{Q, "Q", false, 4}, {S, "S", false, 4}, {W, "W", true, 3}};
    if (int e = check_null(args, 3)) return e;
    int group = 0;
    if (int e = resolve_group(desc, &group)) return e;
    const int tb = desc && desc->trans_b ? 1 : 0;
    if (buf_is_bounds_query(Q) || buf_is_bounds_query(S) || buf_is_bounds_query(W)) return query_w_q_s(args, 2, 0, 1, tb, group);
    if (int e = check_w_q_s(args, 2, 0, 1, tb, group)) return e;
    Q4Params p = {};
    p.N = W->dim[tb ? 1 : 0].extent; p.K = W->dim[tb ? 0 : 1].extent; p.E = W->dim[2].extent;
    if (p.N == 0 || p.K == 0 || p.E == 0) return 0;

    if (int e = rt_ensure_device()) return e;
    const bool sync_after = !(all_resident({Q, S, W}) && tls().async);
    if (int e = check_capture("q4_unpack", sync_after, false)) return e;
    Views vw;
    for (int i = 0; i < 2; ++i, ++vw.n)
        if (int e = rt_input_view(args[i].b, args[i].name, &vw.v[vw.n])) return e;
    if (int e = rt_output_view(W, "W", &vw.v[vw.n])) return e;
    vw.n++;
    p.q = static_cast<uint8_t*>(vw.v[0].ptr);
    p.s = static_cast<uint16_t*>(vw.v[1].ptr);
    p.wout = vw.v[2].ptr;
    p.ldw = W->dim[1].stride; p.bs_w = W->dim[2].stride;
    p.trans_b = tb; p.group = group; p.bf16 = buf_type_word(W) == kBF16;
    if (int e = run_q4("q4_unpack", p, sync_after, q4_unpack_launch)) return e;
    if (int e = rt_finish_output(W, "W", &vw.v[2])) return e;
    return finish_call("q4_unpack", "kernel_Out", sync_after);
}

extern "C" int t2sp_b200_q4_gemv(halide_buffer_t* X, halide_buffer_t* Q, halide_buffer_t* S, halide_buffer_t* index,
                                 halide_buffer_t* Y, const t2sp_q4_desc* desc) {
    Arg args[5] = {{X, "X", false, 2}, {Q, "Q", false, 4}, {S, "S", false, 4}, {Y, "Y", true, 2}, {index, "index", false, 1}};
    if (int e = check_null(args, 4)) return e;   // index may be absent
    const int n_args = index ? 5 : 4;
    int group = 0;
    if (int e = resolve_group(desc, &group)) return e;
    const bool query_index = index && buf_is_bounds_query(index);
    if (buf_is_bounds_query(X) || buf_is_bounds_query(Q) || buf_is_bounds_query(S) || buf_is_bounds_query(Y) || query_index) {
        if (int e = check_query_known(args, n_args)) return e;
        // where X or Y does not say K or N, the most that the packed matrices hold
        int K = 0, N = 0, T = 0, R = 0, E = 1;
        uint32_t t = kBF16;
        if (!buf_is_bounds_query(Q) && Q->dimensions == 4) {
            if (int e = packed_most(args[1], &K, &N)) return e;
            E = Q->dim[3].extent;
        }
        if (!buf_is_bounds_query(S)) t = buf_type_word(S);
        if (!buf_is_bounds_query(X) && X->dimensions == 2) { t = buf_type_word(X); K = X->dim[0].extent; T = R = X->dim[1].extent; }
        if (index && !query_index && index->dimensions == 1) R = index->dim[0].extent;
        if (!buf_is_bounds_query(Y) && Y->dimensions == 2) { N = Y->dim[0].extent; R = Y->dim[1].extent; }
        if (!T) T = R;
        int qe[4], se[4];
        packed_extents(N, K, E, group, qe, se);
        if (buf_is_bounds_query(X)) { int x[2] = {K, T}; fill_query(X, t, 2, x); }
        if (buf_is_bounds_query(Q)) fill_query(Q, kU8, 4, qe);
        if (buf_is_bounds_query(S)) fill_query(S, t, 4, se);
        if (query_index) { int x[1] = {R}; fill_query(index, kI32, 1, x); }
        if (buf_is_bounds_query(Y)) { int x[2] = {N, R}; fill_query(Y, t, 2, x); }
        return 0;
    }
    const uint32_t t = buf_type_word(X);
    if (t != kBF16 && t != kF16) return halide_error_bad_type(nullptr, args[0].role().c_str(), t, kBF16);
    const bool out_f32 = buf_type_word(Y) == kF32;
    if (int e = check_type_dims(args[0], t)) return e;
    if (int e = check_type_dims(args[1], kU8)) return e;
    if (int e = check_type_dims(args[2], t)) return e;
    if (int e = check_type_dims(args[3], out_f32 ? kF32 : t)) return e;
    if (index)
        if (int e = check_type_dims(args[4], kI32)) return e;
    for (int i = 0; i < n_args; ++i)
        if (int e = check_extents_nonneg(args[i])) return e;
    for (int i = 0; i < n_args; ++i)
        if (int e = check_extent_limit(args[i])) return e;
    Q4Params p = {};
    p.K = X->dim[0].extent; p.N = Y->dim[0].extent; p.E = Q->dim[3].extent; p.R = Y->dim[1].extent;
    const int T = X->dim[1].extent;
    if (p.R == 0 || p.N == 0) return 0;
    if (!index && p.E != 1) return constraint("Q.extent.3", p.E, "one matrix where no index is given", 1);
    if (index && index->dim[0].extent != p.R) return constraint("index.extent.0", index->dim[0].extent, "Y.extent.1", p.R);
    if (index && p.R > 1024) return constraint("Y.extent.1", p.R, "at most 1024 rows where an index is given", 1024);
    if (!q4_gemv_fits(p.K, group, p.R, index != nullptr)) return constraint("X.extent.0", p.K, "at most about", 65536);   // a row of x is staged whole in shared memory
    if (T == 0 || p.R % T) return constraint("Y.extent.1", p.R, "a multiple of X.extent.1", T);
    for (int i = 0; i < n_args; ++i)
        if (int e = check_min0(args[i])) return e;
    for (int i = 0; i < n_args; ++i)
        if (int e = check_stride0(args[i])) return e;
    for (int i = 0; i < n_args; ++i)
        if (int e = check_strides(args[i])) return e;
    for (int i = 0; i < n_args; ++i)
        if (int e = check_sizes(args[i])) return e;
    for (int i = 0; i < n_args; ++i)
        if (int e = check_device_address(args[i])) return e;
    int qe[4], se[4];
    packed_extents(p.N, p.K, p.E, group, qe, se);
    if (int e = check_packed(args[1], qe, 16)) return e;
    if (int e = check_packed(args[2], se, 16)) return e;
    for (int i = 0; i < n_args; ++i)
        if (int e = check_host(args[i])) return e;

    if (int e = rt_ensure_device()) return e;
    const bool sync_after = !(all_resident({X, Q, S, Y}) && (!index || all_resident({index})) && tls().async);
    if (int e = check_capture("q4_gemv", sync_after, false)) return e;
    Views vw;
    for (int i = 0; i < 3; ++i, ++vw.n)
        if (int e = rt_input_view(args[i].b, args[i].name, &vw.v[vw.n])) return e;
    if (int e = rt_output_view(Y, "Y", &vw.v[vw.n])) return e;
    vw.n++;
    if (index) {
        if (int e = rt_input_view(index, "index", &vw.v[vw.n])) return e;
        vw.n++;
        if (int e = preload_output(Y, &vw.v[3])) return e;   // rows without a matrix keep their values
    }
    p.x = vw.v[0].ptr;
    p.x_end = static_cast<const uint16_t*>(p.x) + buf_elems_span(X);
    p.ldx = X->dim[1].stride;
    p.q = static_cast<uint8_t*>(vw.v[1].ptr);
    p.s = static_cast<uint16_t*>(vw.v[2].ptr);
    p.y = vw.v[3].ptr;
    p.ldy = Y->dim[1].stride;
    p.index = index ? static_cast<const int*>(vw.v[4].ptr) : nullptr;
    p.per = p.R / T; p.group = group; p.bf16 = t == kBF16; p.out_f32 = out_f32;
    if (int e = run_q4("q4_gemv", p, sync_after, q4_gemv_launch)) return e;
    if (int e = rt_finish_output(Y, "Y", &vw.v[3])) return e;
    return finish_call("q4_gemv", "kernel_Out", sync_after);
}
