// pipe.cuh — asynchronous global->shared staging for persistent kernels:
// 1-D bulk copies (cp.async.bulk, executed by the SM's TMA engine, no
// multicast) completing on shared-memory mbarriers, and bounded waits.
#pragma once

#include "common.cuh"

namespace pbmoe {

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}

// Makes mbarrier initialisation visible to the async (TMA) proxy.
__device__ __forceinline__ void fence_mbar_init() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }

__device__ __forceinline__ void mbar_arrive_expect_tx(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes)
                 : "memory");
}

__device__ __forceinline__ bool mbar_try_wait(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}

// try_wait that may suspend the thread for up to `hint_ns` while the phase
// is incomplete (it resumes as soon as the phase completes).
__device__ __forceinline__ bool mbar_try_wait_hint(uint64_t* bar, uint32_t parity, uint32_t hint_ns) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "r"(hint_ns)
        : "memory");
    return ok != 0;
}

__device__ __forceinline__ uint64_t global_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}

// Wait for phase `parity` of `bar` to complete, giving up after `limit_ns`
// of wall time (returns false; the caller latches an error and winds down).
// Each poll suspends the thread in hardware for up to 20 us, so a waiting
// warp issues a handful of instructions per wait instead of spinning.
__device__ __forceinline__ bool mbar_wait_bounded(uint64_t* bar, uint32_t parity, uint64_t limit_ns) {
    if (mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = global_ns();
    while (!mbar_try_wait_hint(bar, parity, 20000u)) {
        if (global_ns() - t0 > limit_ns) return false;
    }
    return true;
}

// Contiguous copy global -> shared through the TMA unit (both addresses 16-byte
// aligned, size a multiple of 16), completing as transaction bytes on `bar`.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                     smem_u32(dst)),
                 "l"(src), "r"(bytes), "r"(smem_u32(bar))
                 : "memory");
}

// 16-byte asynchronous copy global -> shared through L2 (no L1 allocation).
// Unlike a bulk copy, each is a plain LSU request, so thousands of small
// row pieces per stage cost no per-copy TMA setup, and the destination may
// be any padded layout.
__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}

// 4-byte asynchronous copy global -> shared (both addresses 4-byte aligned).
__device__ __forceinline__ void cp_async4(void* dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
// Close this thread's current group of cp.async copies; wait until at most N
// of its groups are still in flight.
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait_group() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Arrive on `bar` once every cp.async this thread issued so far has landed.
// The arrival is not added to the pending count: the barrier's expected
// count must include one arrival per issuing thread and phase.
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// Wait until this thread's own cp.async copies have landed.
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// Named CTA barriers (ids 1..15; 0 is __syncthreads) for warp-specialised
// producer/consumer hand-offs. `count` is the number of participating threads
// (a multiple of 32): arrive() never blocks, sync() waits for the count.
__device__ __forceinline__ void named_sync(int id, int count) {
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(count) : "memory");
}
// sync() that also returns whether any participant's `vote` was set.
__device__ __forceinline__ bool named_sync_or(int id, int count, bool vote) {
    uint32_t r;
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.u32 p, %3, 0;\n barrier.cta.red.or.pred q, %1, %2, p;\n"
        " selp.u32 %0, 1, 0, q;\n}\n"
        : "=r"(r)
        : "r"(id), "r"(count), "r"(vote ? 1u : 0u)
        : "memory");
    return r != 0;
}
__device__ __forceinline__ void named_arrive(int id, int count) {
    asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(count) : "memory");
}

// Wall-time bound of every pipeline wait (a healthy wait is microseconds).
constexpr uint64_t kPipeWaitNs = 2000000000ull;

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// Bounded wait that also stops when another role of the CTA has aborted.
__device__ __forceinline__ bool wait_or_abort(uint64_t* bar, uint32_t parity, volatile uint32_t* abort_flag,
                                              uint32_t* status) {
    if (mbar_try_wait(bar, parity)) return true;
    if (mbar_try_wait_hint(bar, parity, 20000u)) return true;  // no timer read in a healthy wait
    const uint64_t t0 = global_ns();
    while (!mbar_try_wait_hint(bar, parity, 20000u)) {
        if (*abort_flag) return false;
        if (global_ns() - t0 > kPipeWaitNs) {
            *abort_flag = 1u;
            if (status) atomicOr(status, PBMOE_DEV_ERR_PIPE_TIMEOUT);
            return false;
        }
    }
    return true;
}

// Bounded wait for roles off the critical path (epilogue, loader): polls with
// a short sleep in between, so the waiting warp does not take issue slots
// from the dequant warp on its scheduler.
__device__ __forceinline__ bool wait_or_abort_lazy(uint64_t* bar, uint32_t parity, volatile uint32_t* abort_flag,
                                                   uint32_t* status) {
    if (mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = global_ns();
    for (;;) {
        __nanosleep(256);
        if (mbar_try_wait(bar, parity)) return true;
        if (*abort_flag) return false;
        if (global_ns() - t0 > kPipeWaitNs) {
            *abort_flag = 1u;
            if (status) atomicOr(status, PBMOE_DEV_ERR_PIPE_TIMEOUT);
            return false;
        }
    }
}

// A wait decided by lane 0 and broadcast, so the warp stays converged for the
// warp-collective operations that follow.
template <bool kLazy>
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile uint32_t* abort_flag,
                                          uint32_t* status) {
    bool ok = false;
    if ((threadIdx.x & 31) == 0)
        ok = kLazy ? wait_or_abort_lazy(bar, parity, abort_flag, status) : wait_or_abort(bar, parity, abort_flag, status);
    return __shfl_sync(kFull, ok ? 1u : 0u, 0) != 0u;
}

}  // namespace pbmoe
