// Wrappers of the instructions that kernels on the 5th-generation tensor cores are made of: mbarriers, bulk-tensor copies, tensor
// memory, and the descriptors of tcgen05.mma operands in shared memory.
#pragma once
#include <cuda.h>   // CUtensorMap and the types of cuTensorMapEncodeTiled (the entry point is looked up at run time)

#include "common.cuh"

namespace ojx {

__device__ __forceinline__ unsigned tc_smem(const void* p) { return static_cast<unsigned>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void tc_bar_init(unsigned bar, unsigned count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void tc_bar_arrive(unsigned bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void tc_bar_expect(unsigned bar, unsigned bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

// Waits of a warp for a phase: one look where it is there already, else as bar_wait waits.  False: it ran out.
__device__ __forceinline__ bool tc_wait(unsigned bar, unsigned parity, unsigned gone, long long clocks = kBarClocks) {
    unsigned done;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    return __all_sync(0xffffffffu, done) || __all_sync(0xffffffffu, bar_wait(bar, parity, gone, clocks));
}
// Asks for a CTA of the grid that has not begun, to do its work in its place: 16 bytes at `to` and on `bar` (whose transaction count
// the caller raises); then its number, or -1 where there is none any more (after which nothing may be asked again).
__device__ __forceinline__ void tc_steal(unsigned to, unsigned bar) {
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(to), "r"(bar) : "memory");
}
__device__ __forceinline__ int tc_stolen(unsigned from) {
    int cta;
    asm volatile(
        "{\n\t.reg .b128 h;\n\t.reg .pred p;\n\tld.shared.b128 h, [%1];\n\tmov.u32 %0, -1;\n\t"
        "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\t"
        "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %0, h;\n\t}"
        : "=r"(cta)
        : "r"(from)
        : "memory");
    return cta;
}
// A place in a ring of N stages and the parity of its next phase.
template <int N>
struct TcRing {
    int slot;
    unsigned parity;
    __device__ __forceinline__ void next(int by) {
        slot += by;
        if (slot >= N) { slot -= N; parity ^= 1u; }
    }
};

// Box of a 3-dimensional tensor map to shared memory; x in elements, a multiple of 16 bytes.
__device__ __forceinline__ void tc_load3(unsigned to, const CUtensorMap* map, int x, int y, int z, unsigned bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(to),
                 "l"(reinterpret_cast<unsigned long long>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
                 : "memory");
}

// Operand in shared memory with the 128-byte swizzle.  K-major: rows of 64 16-bit elements (128 bytes), eight rows 1024 bytes; a step
// of 16 along K is 32 bytes.  MN-major: the rows are steps along K, the 64 elements lie along M or N; `next`: bytes to the next 64.
__device__ __forceinline__ unsigned long long tc_desc(unsigned addr, unsigned next = 16) {
    return (unsigned long long)((addr >> 4) & 0x3fff) | (unsigned long long)((next >> 4) & 0x3fff) << 16 | (unsigned long long)(1024 >> 4) << 32 |
           (unsigned long long)1 << 46 | (unsigned long long)2 << 61;
}

// The same `bytes` further on (whole multiples of 16; shared memory ends before the address field does).
__device__ __forceinline__ unsigned long long tc_at(unsigned long long desc, int bytes) { return desc + (unsigned)(bytes >> 4); }

// Instruction descriptor: fp32 sums, operands of 16 bits (bf16, or fp16), M = 128; kMnB: the B operand is MN-major.
template <bool kBf16, bool kMnB>
__device__ __forceinline__ constexpr unsigned tc_idesc(int n) {
    return 1u << 4 | (kBf16 ? 1u << 7 | 1u << 10 : 0u) | (kMnB ? 1u << 16 : 0u) | (unsigned)(n >> 3) << 17 | (unsigned)(128 >> 4) << 24;
}

// Products and commits are issued by whole warps, of which one lane (`lead`) acts: descriptors and addresses that are the same in all
// lanes stay in uniform registers, where the instruction takes them from.  Issued from a branch of one lane they were moved there
// for every product, 126 to 180 clocks each.
__device__ __forceinline__ unsigned tc_lead() {
    unsigned lead;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(lead));
    return lead;
}
__device__ __forceinline__ void tc_mma(unsigned lead, unsigned d, unsigned long long a, unsigned long long b, unsigned idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"((unsigned)add), "r"(lead)
        : "memory");
}
// The A operand in tensor memory: a row per lane, two 16-bit elements per column.
__device__ __forceinline__ void tc_mma_ts(unsigned lead, unsigned d, unsigned a, unsigned long long b, unsigned idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"((unsigned)add), "r"(lead)
        : "memory");
}
// Arrives at `bar` when the products issued so far are done.
__device__ __forceinline__ void tc_commit(unsigned lead, unsigned bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar),
        "r"(lead)
        : "memory");
}

#define OJX_R8(v, i) "=r"((v)[i]), "=r"((v)[i + 1]), "=r"((v)[i + 2]), "=r"((v)[i + 3]), "=r"((v)[i + 4]), "=r"((v)[i + 5]), "=r"((v)[i + 6]), "=r"((v)[i + 7])
#define OJX_I8(v, i) "r"((v)[i]), "r"((v)[i + 1]), "r"((v)[i + 2]), "r"((v)[i + 3]), "r"((v)[i + 4]), "r"((v)[i + 5]), "r"((v)[i + 6]), "r"((v)[i + 7])
// 32 columns of the warp's 32 lanes (all threads of the warp, whose lanes are 32 * (warp % 4) on); wait before using them.
__device__ __forceinline__ void tc_ld32(unsigned addr, unsigned* v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, "
        "%22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : OJX_R8(v, 0), OJX_R8(v, 8), OJX_R8(v, 16), OJX_R8(v, 24)
        : "r"(addr));
}
__device__ __forceinline__ void tc_st32(unsigned addr, const unsigned* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, "
        "%21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::OJX_I8(v, 0), OJX_I8(v, 8), OJX_I8(v, 16), OJX_I8(v, 24), "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tc_st16(unsigned addr, const unsigned* v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::OJX_I8(v, 0), OJX_I8(v, 8), "r"(addr)
                 : "memory");
}
__device__ __forceinline__ unsigned tc_ld1(unsigned addr) {
    unsigned v;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(v) : "r"(addr));
    return v;
}
#define OJX_P8(v, i) "+r"((v)[i]), "+r"((v)[i + 1]), "+r"((v)[i + 2]), "+r"((v)[i + 3]), "+r"((v)[i + 4]), "+r"((v)[i + 5]), "+r"((v)[i + 6]), "+r"((v)[i + 7])
// Keeps the uses of loaded columns behind the wait for them.
__device__ __forceinline__ void tc_pin32(unsigned* v) { asm volatile("" : OJX_P8(v, 0), OJX_P8(v, 8), OJX_P8(v, 16), OJX_P8(v, 24)); }
#undef OJX_R8
#undef OJX_I8
#undef OJX_P8
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// A 3-dimensional tensor of 16-bit elements, strides in elements; false where the driver does not take it.
inline bool tc_map3(CUtensorMap* map, bool bf16, const void* base, unsigned long long d0, unsigned long long d1, unsigned long long d2,
                    unsigned long long s1, unsigned long long s2, unsigned b0, unsigned b1, unsigned b2) {
    using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static Encode encode = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) {
            cudaGetLastError();
            p = nullptr;
        }
        return reinterpret_cast<Encode>(p);
    }();
    if (!encode) return false;
    const cuuint64_t dims[3] = {d0, d1, d2}, strides[2] = {s1 * 2, s2 * 2};
    const cuuint32_t box[3] = {b0, b1, b2}, step[3] = {1, 1, 1};
    return encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base), dims, strides, box, step,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace ojx
