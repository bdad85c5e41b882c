// Launches of the attention over a paged cache: one kernel per type, dimension and heads of a pass, each with its own registers, for
// the plain and the best-effort flavour.  Like the tcgen05 kernels it is not hosted by the dispatcher: padding launches ranges of its
// blocks beside the real-time kernel.
#include "paged_attention.cuh"
#include "tc_common.cuh"

#include <cstring>
#include <string>

#include "registry.h"

namespace reef {

extern __shared__ __align__(16) unsigned char reef_paged_smem[];

// flag: best-effort flavour, else null; slot: completion counter, may be null; blocks [first, first + gridDim.x) of the kernel
template <class E, int BLOCKS>
__global__ void __launch_bounds__(kThreads, BLOCKS) k_paged_attention(const __grid_constant__ KTask t, int first, const int* flag, int* slot,
                                                                 unsigned long long* stamps) {
    const int up = flag != nullptr && threadIdx.x == 0 ? ld_flag(flag) : 0;
    pdl_prologue();
    const bool go = flag == nullptr || !__syncthreads_or(up);
    const bool done = go && paged_attention_body<E>(t, first + blockIdx.x, reef_paged_smem, flag);
    if (slot == nullptr) return;
    const int stopped = __syncthreads_or(done ? 0 : 1);
    if (threadIdx.x == 0) {
        if (!stopped) {
            red_relaxed_gpu_add(slot, 1);
        } else if (stamps != nullptr) {
            unsigned long long now;
            asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
            atomicMin(&stamps[0], now);
            atomicMax(&stamps[1], now);
        }
    }
}

template <class C, int D>
struct PagedFns {
    static const void* of(int gb) {
        return gb == 1 ? (const void*)k_paged_attention<PagedSimt<C, D, 1>, 2>
             : gb == 2 ? (const void*)k_paged_attention<PagedSimt<C, D, 2>, 2>
             : gb == 4 ? (const void*)k_paged_attention<PagedMma<C, D, 4>, 1>
             : gb == 8 ? (const void*)k_paged_attention<PagedMma<C, D, 8>, 1> : nullptr;
    }
};
template <int D, int GB>
static const void* paged_fp32() {
    if constexpr (D == 256 && GB > 4) return nullptr;
    else return (const void*)k_paged_attention<PagedSimt<float, D, GB>, 2>;
}
template <int D>
struct PagedFns<float, D> {
    static const void* of(int gb) {
        switch (gb) {
            case 1: return paged_fp32<D, 1>();
            case 2: return paged_fp32<D, 2>();
            case 3: return paged_fp32<D, 3>();
            case 4: return paged_fp32<D, 4>();
            case 5: return paged_fp32<D, 5>();
            case 6: return paged_fp32<D, 6>();
            case 8: return paged_fp32<D, 8>();
            default: return nullptr;
        }
    }
};
template <class C>
static const void* paged_fn_dim(int d, int gb) {
    return d == 64 ? PagedFns<C, 64>::of(gb) : d == 128 ? PagedFns<C, 128>::of(gb) : d == 256 ? PagedFns<C, 256>::of(gb) : nullptr;
}
static const void* paged_fn(const PagedP& p) {
    return p.kt == KT_FP32 ? paged_fn_dim<float>(p.d, p.gb) : p.kt == KT_BF16 ? paged_fn_dim<__nv_bfloat16>(p.d, p.gb) : paged_fn_dim<__half>(p.d, p.gb);
}

// on the current device, ahead of the first launch there: a part of what reef_kernel_prepare does once
int paged_prepare_device() {
    for (int kt = KT_FP32; kt <= KT_FP16; kt++)
        for (int d = 64; d <= 256; d *= 2)
            for (int gb = 1; gb <= 8; gb++) {
                PagedP p;
                p.kt = kt; p.d = d; p.gb = gb;
                const void* fn = paged_fn(p);
                if (fn == nullptr) continue;
                cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, paged_attention_smem(p));
                if (e == cudaSuccess) e = cudaFuncSetAttribute(fn, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
                if (e != cudaSuccess) {
                    set_error(std::string("cudaFuncSetAttribute(paged attention): ") + cudaGetErrorString(e));
                    return REEF_FAIL;
                }
            }
    return REEF_SUCC;
}

int paged_launch(const KTask& t, uint32_t smem, cudaStream_t st, const int* flag, int* slot, int first, int count) {
    if (count < 0) count = t.nblocks - first;
    if (first < 0 || count <= 0 || first + count > t.nblocks) {
        set_error("paged attention: block range outside the kernel");
        return REEF_OUT_OF_RANGE;
    }
    unsigned long long* stamps = flag != nullptr ? preempt_stamps_ptr() : nullptr;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(count);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    void* args[] = {const_cast<KTask*>(&t), &first, (void*)&flag, (void*)&slot, (void*)&stamps};
    const cudaError_t e = cudaLaunchKernelExC(&cfg, paged_fn(t.p.paged), args);
    if (e != cudaSuccess) {
        set_error(std::string("cudaLaunchKernelExC(paged attention): ") + cudaGetErrorString(e));
        return REEF_FAIL;
    }
    return REEF_SUCC;
}

int paged_func_attrs(const PagedP& p, uint32_t smem, cudaFuncAttributes* fa, int* occ) {
    cudaError_t e = cudaFuncGetAttributes(fa, paged_fn(p));
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(occ, paged_fn(p), kThreads, smem);
    if (e != cudaSuccess) {
        set_error(std::string("cudaFuncGetAttributes(paged attention): ") + cudaGetErrorString(e));
        return REEF_FAIL;
    }
    return REEF_SUCC;
}

}  // namespace reef
