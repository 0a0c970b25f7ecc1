// Entry points of the grouped products: argument validation in the order of the other entries (ops.cpp), then one
// launch over the rows of all groups. The group boundaries stay on the device: nothing here reads them.
#include "grouped.h"
#include "op_common.h"

using namespace t2sp;

namespace t2sp {
namespace {

int check_offsets(const Arg& a) {
    if (a.b->dim[0].extent < 1) return constraint("offsets.extent.0", a.b->dim[0].extent, "groups + 1", 1);
    if (a.b->dim[0].extent > kMaxGroups + 1)
        return constraint("offsets.extent.0", a.b->dim[0].extent, "at most groups + 1", kMaxGroups + 1);
    return 0;
}

// A matrix operand as TMA reads it: 16-byte aligned base, strides that are multiples of 16 bytes.
struct Operand {
    char* ptr;
    int64_t ld, bs;              // elements between rows and between matrices
    int inner, rows, matrices;
    bool fits() const {
        return !(reinterpret_cast<uintptr_t>(ptr) & 15) && (rows <= 1 || ld % 8 == 0) && (matrices <= 1 || bs % 8 == 0);
    }
};

// Copies operands that TMA cannot read in place into scratch memory with padded rows.
int fit_operands(Views& vw, Operand* a, Operand* b) {
    Repack jobs[2];
    int count = 0;
    for (Operand* o : {a, b}) {
        if (!o || o->fits()) continue;
        const int64_t ld = (int64_t(o->inner) + 7) / 8 * 8;
        void* q = rt_alloc(size_t(ld) * o->rows * o->matrices * 2);
        if (!q) return halide_error_code_device_malloc_failed;
        vw.v[vw.n].ptr = q; vw.v[vw.n].borrowed = false; vw.n++;
        jobs[count++] = {reinterpret_cast<const uint16_t*>(o->ptr), static_cast<uint16_t*>(q), o->ld, o->bs, ld, o->inner, o->rows, o->matrices, 0};
        o->ptr = static_cast<char*>(q);
        o->ld = ld;
        o->bs = ld * o->rows;
    }
    if (count == 0) return 0;
    if (repack16_launch(jobs, count, rt_stream()) != cudaSuccess) {
        cudaGetLastError();
        return halide_error_code_device_run_failed;
    }
    rt_count_launch(1);
    return 0;
}

bool encode(CUtensorMap* map, uint32_t type, const Operand& o, int rank, uint32_t box_inner, uint32_t box_rows) {
    // strides of dimensions of one element are never used, but have to be multiples of 16 bytes
    const uint64_t ld = o.rows > 1 ? uint64_t(o.ld) * 2 : (uint64_t(o.inner) * 2 + 15) / 16 * 16;
    const uint64_t bs = o.matrices > 1 ? uint64_t(o.bs) * 2 : ld * o.rows;
    const uint64_t dims[3] = {uint64_t(o.inner), uint64_t(o.rows), uint64_t(o.matrices)}, str[3] = {2, ld, bs};
    const uint32_t box[3] = {box_inner, box_rows, 1};
    return rt_encode_tmap(map, type == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank, o.ptr, dims,
                          str, box);
}

// Lowering and launch, with the timing and the error report of the other operators. `p_op` holds the columns n (B, or D),
// `q_op` the rows (A).
int run_grouped(const char* who, int mode, uint32_t type, uint32_t out, GroupedParams& p, Operand p_op, Operand q_op, Views& vw,
                bool sync_after) {
    const int out_kind = out == kF32 ? GR_OUT_F32 : (out == kBF16 ? GR_OUT_BF16 : GR_OUT_F16);
    const bool in_place = !p_op.fits() && grouped_warps_worthwhile(mode, out_kind, p);
    if (int e = check_capture(who, false, (!p_op.fits() && !in_place) || !q_op.fits())) return e;
    cudaStream_t s = rt_stream();
    p.status = rt_status_word();
    p.wait_cycles = rt_env().wait_cycles;
    p.skip_stage = rt_env().test_skip_stage;
    p.bf16 = type == kBF16;
    if (sync_after) cudaEventRecord(rt_event(0), s);
    GroupedMaps maps;
    memset(&maps, 0, sizeof(maps));
    if (p.K > 0 && p.rows > 0) {   // else nothing is read
        if (in_place) {
            p.b_src = reinterpret_cast<const uint16_t*>(p_op.ptr);
            p.b_end = p.b_src + (p_op.matrices - 1) * p_op.bs + (p_op.rows - 1) * p_op.ld + p_op.inner;
            p.b_ld = p_op.ld;
            p.b_bs = p_op.bs;
        }
        if (int e = fit_operands(vw, in_place ? nullptr : &p_op, &q_op)) return e;
        bool ok = (in_place || encode(&maps.p, type, p_op, 3, 64, mode == GR_FWD_K ? 128 : 64)) &&
                  encode(&maps.q[0], type, q_op, 2, 64, mode == GR_GRAD ? 64 : 128);
        if (mode == GR_GRAD) {
            ok = ok && encode(&maps.q[1], type, p_op, 3, 64, 16) && encode(&maps.q[2], type, q_op, 2, 64, 16);
        } else {
            for (int b = 1; b < 4; ++b) ok = ok && encode(&maps.q[b], type, q_op, 2, 64, 128 >> b);
        }
        if (!ok) return tma_unsupported(mode == GR_GRAD ? "A or D" : "A or B");
    }
    const cudaError_t e = grouped_launch(mode, out_kind, p, maps, s);
    if (e != cudaSuccess) {
        fprintf(stderr, "t2sp_b200: %s: kernel launch failed: %s\n", who, cudaGetErrorString(e));
        return halide_error_code_device_run_failed;
    }
    rt_count_launch(1);
    if (sync_after) cudaEventRecord(rt_event(1), s);
    return 0;
}

}  // namespace
}  // namespace t2sp

extern "C" int t2sp_b200_grouped_gemm(halide_buffer_t* A, halide_buffer_t* B, halide_buffer_t* offsets, halide_buffer_t* C,
                                      const t2sp_grouped_desc* desc) {
    Arg args[4] = {{A, "A", false, 2}, {B, "B", false, 3}, {offsets, "offsets", false, 1}, {C, "C", true, 2}};
    if (int e = check_null(args, 4)) return e;
    const int tb = desc && desc->trans_b ? 1 : 0;
    if (buf_is_bounds_query(A) || buf_is_bounds_query(B) || buf_is_bounds_query(offsets) || buf_is_bounds_query(C)) {
        if (int e = check_query_known(args, 4)) return e;
        if (!buf_is_bounds_query(offsets) && offsets->dimensions == 1)
            if (int e = check_offsets(args[2])) return e;
        int K = 0, M = 0, N = 0, E = 0;
        if (!buf_is_bounds_query(A) && A->dimensions == 2) { K = A->dim[0].extent; M = A->dim[1].extent; }
        if (!buf_is_bounds_query(B) && B->dimensions == 3) {
            N = B->dim[tb ? 1 : 0].extent;
            E = B->dim[2].extent;
            if (!K) K = B->dim[tb ? 0 : 1].extent;
        }
        if (!buf_is_bounds_query(offsets) && offsets->dimensions == 1 && !E) E = offsets->dim[0].extent - 1;
        if (!buf_is_bounds_query(C) && C->dimensions == 2) {
            if (!N) N = C->dim[0].extent;
            if (!M) M = C->dim[1].extent;
        }
        const uint32_t t = !buf_is_bounds_query(A) ? buf_type_word(A) : (!buf_is_bounds_query(B) ? buf_type_word(B) : kBF16);
        if (buf_is_bounds_query(A)) { int x[2] = {K, M}; fill_query(A, t, 2, x); }
        if (buf_is_bounds_query(B)) { int x[3] = {tb ? K : N, tb ? N : K, E}; fill_query(B, t, 3, x); }
        if (buf_is_bounds_query(offsets)) { int x[1] = {E + 1}; fill_query(offsets, kI32, 1, x); }
        if (buf_is_bounds_query(C)) { int x[2] = {N, M}; fill_query(C, t, 2, x); }
        return 0;
    }
    const uint32_t in_t = buf_type_word(A);
    if (in_t != kBF16 && in_t != kF16) return halide_error_bad_type(nullptr, args[0].role().c_str(), in_t, kBF16);
    const bool out_f32 = buf_type_word(C) == kF32;
    if (int e = check_type_dims(args[0], in_t)) return e;
    if (int e = check_type_dims(args[1], in_t)) return e;
    if (int e = check_type_dims(args[2], kI32)) return e;
    if (int e = check_type_dims(args[3], out_f32 ? kF32 : in_t)) return e;
    for (auto& a : args)
        if (int e = check_extents_nonneg(a)) return e;
    for (auto& a : args)
        if (int e = check_extent_limit(a)) return e;
    const int K = A->dim[0].extent, M = A->dim[1].extent, N = B->dim[tb ? 1 : 0].extent, E = B->dim[2].extent;
    if (B->dim[tb ? 0 : 1].extent != K)
        return constraint(tb ? "B.extent.0" : "B.extent.1", B->dim[tb ? 0 : 1].extent, "A.extent.0", K);
    if (int e = check_offsets(args[2])) return e;
    if (offsets->dim[0].extent != E + 1) return constraint("offsets.extent.0", offsets->dim[0].extent, "B.extent.2 + 1", E + 1);
    for (int i = 0; i < 3; ++i)
        if (int e = check_min0(args[i])) return e;
    if (int e = check_covers(args[3], 0, N)) return e;
    if (int e = check_covers(args[3], 1, M)) return e;
    for (auto& a : args)
        if (int e = check_stride0(a)) return e;
    for (auto& a : args)
        if (int e = check_strides(a)) return e;
    for (auto& a : args)
        if (int e = check_sizes(a)) return e;
    for (auto& a : args)
        if (int e = check_device_address(a)) return e;
    for (auto& a : args)
        if (int e = check_host(a)) return e;
    if (M == 0 || N == 0 || E == 0) return 0;

    if (int e = rt_ensure_device()) return e;
    const bool sync_after = !(all_resident({A, B, offsets, C}) && tls().async);
    if (int e = check_capture("grouped_gemm", sync_after, false)) return e;
    Views vw;
    for (int i = 0; i < 3; ++i, ++vw.n)
        if (int e = rt_input_view(args[i].b, args[i].name, &vw.v[vw.n])) return e;
    if (int e = rt_output_view(C, "C", &vw.v[vw.n])) return e;
    vw.n++;
    if (int e = preload_output(C, &vw.v[3])) return e;   // rows outside the groups keep their values
    GroupedParams p = {};
    p.offsets = static_cast<const int*>(vw.v[2].ptr);
    p.c = static_cast<char*>(vw.v[3].ptr) + origin_offset(C) * (out_f32 ? 4 : 2);
    p.ldc = C->dim[1].stride;
    p.rows = M; p.E = E; p.K = K; p.N = N;
    const Operand b = {static_cast<char*>(vw.v[1].ptr), B->dim[1].stride, B->dim[2].stride, B->dim[0].extent, B->dim[1].extent, E};
    const Operand a = {static_cast<char*>(vw.v[0].ptr), A->dim[1].stride, 0, K, M, 1};
    if (int e = run_grouped("grouped_gemm", tb ? GR_FWD_K : GR_FWD_MN, in_t, out_f32 ? kF32 : in_t, p, b, a, vw, sync_after)) return e;
    if (int e = rt_finish_output(C, "C", &vw.v[3])) return e;
    return finish_call("grouped_gemm", "kernel_Out", sync_after);
}

extern "C" int t2sp_b200_grouped_gemm_grad(halide_buffer_t* A, halide_buffer_t* D, halide_buffer_t* offsets, halide_buffer_t* G) {
    Arg args[4] = {{A, "A", false, 2}, {D, "D", false, 2}, {offsets, "offsets", false, 1}, {G, "G", true, 3}};
    if (int e = check_null(args, 4)) return e;
    if (buf_is_bounds_query(A) || buf_is_bounds_query(D) || buf_is_bounds_query(offsets) || buf_is_bounds_query(G)) {
        if (int e = check_query_known(args, 4)) return e;
        if (!buf_is_bounds_query(offsets) && offsets->dimensions == 1)
            if (int e = check_offsets(args[2])) return e;
        int K = 0, M = 0, N = 0, E = 0;
        if (!buf_is_bounds_query(A) && A->dimensions == 2) { K = A->dim[0].extent; M = A->dim[1].extent; }
        if (!buf_is_bounds_query(D) && D->dimensions == 2) { N = D->dim[0].extent; if (!M) M = D->dim[1].extent; }
        if (!buf_is_bounds_query(G) && G->dimensions == 3) {
            if (!N) N = G->dim[0].extent;
            if (!K) K = G->dim[1].extent;
            E = G->dim[2].extent;
        }
        if (!buf_is_bounds_query(offsets) && offsets->dimensions == 1 && !E) E = offsets->dim[0].extent - 1;
        const uint32_t t = !buf_is_bounds_query(A) ? buf_type_word(A) : (!buf_is_bounds_query(D) ? buf_type_word(D) : kBF16);
        if (buf_is_bounds_query(A)) { int x[2] = {K, M}; fill_query(A, t, 2, x); }
        if (buf_is_bounds_query(D)) { int x[2] = {N, M}; fill_query(D, t, 2, x); }
        if (buf_is_bounds_query(offsets)) { int x[1] = {E + 1}; fill_query(offsets, kI32, 1, x); }
        if (buf_is_bounds_query(G)) { int x[3] = {N, K, E}; fill_query(G, t, 3, x); }
        return 0;
    }
    const uint32_t in_t = buf_type_word(A);
    if (in_t != kBF16 && in_t != kF16) return halide_error_bad_type(nullptr, args[0].role().c_str(), in_t, kBF16);
    const bool out_f32 = buf_type_word(G) == kF32;
    if (int e = check_type_dims(args[0], in_t)) return e;
    if (int e = check_type_dims(args[1], in_t)) return e;
    if (int e = check_type_dims(args[2], kI32)) return e;
    if (int e = check_type_dims(args[3], out_f32 ? kF32 : in_t)) return e;
    for (auto& a : args)
        if (int e = check_extents_nonneg(a)) return e;
    for (auto& a : args)
        if (int e = check_extent_limit(a)) return e;
    const int K = A->dim[0].extent, M = A->dim[1].extent, N = D->dim[0].extent;
    if (D->dim[1].extent != M) return constraint("D.extent.1", D->dim[1].extent, "A.extent.1", M);
    if (int e = check_offsets(args[2])) return e;
    const int E = offsets->dim[0].extent - 1;
    for (int i = 0; i < 3; ++i)
        if (int e = check_min0(args[i])) return e;
    if (int e = check_covers(args[3], 0, N)) return e;
    if (int e = check_covers(args[3], 1, K)) return e;
    if (int e = check_covers(args[3], 2, E)) return e;
    for (auto& a : args)
        if (int e = check_stride0(a)) return e;
    for (auto& a : args)
        if (int e = check_strides(a)) return e;
    for (auto& a : args)
        if (int e = check_sizes(a)) return e;
    for (auto& a : args)
        if (int e = check_device_address(a)) return e;
    for (auto& a : args)
        if (int e = check_host(a)) return e;
    if (K == 0 || N == 0 || E == 0) return 0;

    if (int e = rt_ensure_device()) return e;
    const bool sync_after = !(all_resident({A, D, offsets, G}) && tls().async);
    if (int e = check_capture("grouped_gemm_grad", sync_after, false)) return e;
    Views vw;
    for (int i = 0; i < 3; ++i, ++vw.n)
        if (int e = rt_input_view(args[i].b, args[i].name, &vw.v[vw.n])) return e;
    if (int e = rt_output_view(G, "G", &vw.v[vw.n])) return e;
    vw.n++;
    if (int e = preload_output(G, &vw.v[3])) return e;   // what G holds beyond (N, K, E) keeps its values
    GroupedParams p = {};
    p.offsets = static_cast<const int*>(vw.v[2].ptr);
    p.c = static_cast<char*>(vw.v[3].ptr) + origin_offset(G) * (out_f32 ? 4 : 2);
    p.ldc = G->dim[1].stride;
    p.bs_c = G->dim[2].stride;
    p.rows = M; p.E = E; p.K = K; p.N = N;
    const Operand d = {static_cast<char*>(vw.v[1].ptr), D->dim[1].stride, 0, N, M, 1};
    const Operand a = {static_cast<char*>(vw.v[0].ptr), A->dim[1].stride, 0, K, M, 1};
    if (int e = run_grouped("grouped_gemm_grad", GR_GRAD, in_t, out_f32 ? kF32 : in_t, p, d, a, vw, sync_after)) return e;
    if (int e = rt_finish_output(G, "G", &vw.v[3])) return e;
    return finish_call("grouped_gemm_grad", "kernel_Out", sync_after);
}
