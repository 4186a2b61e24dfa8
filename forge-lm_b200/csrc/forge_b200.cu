// forge_b200.cu — runtime and C ABI of libforge_b200.so (sm_100a).
//
// Host-side structure:
//   fb2_model   : per-device fp32 weight copies (one contiguous allocation).
//   fb2_session : per-device DeviceSession (stream, KV cache, histories,
//                 activation buffers, captured decode-step graph).
// The token loop (Sampler.Generate, src/LLM.Core/Inference/Sampler.cs:78-109)
// runs as: one prefill of every prompt window, then per step a CUDA-graph
// replay of the KV-cached decode step for the slots whose window still fits
// the context, a full re-prefill for the slots whose window slides
// (Sampler.cs:93-94), and the on-device sampler for all slots.
#include <cuda_runtime.h>

#include <algorithm>
#include <array>
#include <unordered_map>
#include <atomic>
#include <cctype>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <mutex>
#include <stdexcept>
#include <string>
#include <thread>
#include <vector>

#include "../../include/forge_b200.h"
#include "../../include/forge_b200_testing.h"
#include "capi.cuh"
#include "dotnet_random.hpp"
#include "kernels.cuh"
#include "sampler.cuh"
#include "decode_mega.cuh"
#include "gemm_tc.cuh"
#include "attn_tc.cuh"
#include "forgemodel.hpp"
#include "tokenizer.hpp"

#include <cudaTypedefs.h>

using namespace fb2;

namespace {
// Test hook (fb2_test_fail_alloc): the g_fail_alloc_at-th device allocation
// from now fails as if the device were out of memory; counted over the
// process, 0 = off.
std::atomic<long long> g_alloc_count{0};
std::atomic<long long> g_fail_alloc_at{0};

template <class T>
T* dalloc(size_t n) {
    void* p = nullptr;
    if (n == 0) n = 1;
    const long long k = ++g_alloc_count;
    const long long at = g_fail_alloc_at.load();
    if (at > 0 && k == at) {
        g_fail_alloc_at = 0;
        fail(FB2_OUT_OF_MEMORY, "cudaMalloc: out of memory (injected by fb2_test_fail_alloc)");
    }
    CK(cudaMalloc(&p, n * sizeof(T)));
    return static_cast<T*>(p);
}
template <class T>
void dfree(T*& p) {
    if (p) cudaFree(p);
    p = nullptr;
}

inline int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }

constexpr int kMaxGemvRows = 16;
constexpr int kTcSplitMax = 32;  // k splits of the decode tensor-core GEMM
constexpr int kMaxChunkSlots = 64;  // sequences per prefill chunk (head scratch rows)
constexpr int kGemvMaxKChunk = 256;
}  // namespace

// ---------------------------------------------------------------------------
// model
// ---------------------------------------------------------------------------
struct LayerW {
    const float *ln1_w, *ln1_b, *qkv_w, *qkv_b, *proj_w, *proj_b, *ln2_w, *ln2_b, *fc_w, *fc_b, *mproj_w, *mproj_b;
};

struct DeviceModel {
    int device = 0;
    int sm_count = 148;
    float* blob = nullptr;
    std::vector<const float*> p;
    std::vector<LayerW> layers;
    const float *tok_emb = nullptr, *pos_emb = nullptr, *lnf_w = nullptr, *lnf_b = nullptr;
    // persistent decode kernel: projections re-laid as per-CTA column strips
    bool mk_ok = false;
    int mk_nW = 0;
    // head-cluster layout of the persistent kernel: clusters of mk_cs CTAs,
    // mk_nhead = H * mk_cs attention CTAs, the rest run the MLP
    bool mk_hc = false;
    int mk_cs = 1, mk_nhead = 0;
    float* relaid = nullptr;
    float* mk_fold = nullptr;  // head-cluster layout: folded-LayerNorm (S, B) per qkv / fc column
    MkLayer* d_mk_layers = nullptr;
    // tensor-core GEMM: TF32 hi/lo halves of the four projections per layer
    // (qkv, proj, fc, mlp proj) and their TMA descriptors
    bool tc_ok = false;
    // prefill attention on the tensor cores (head_dim 64; FORGE_B200_ATTN=simt
    // keeps the SIMT kernel)
    bool attn_tc = false;
    float* tc_blob = nullptr;
    // FB2_WEIGHTS_BF16: the projections and tok_emb are rounded to bf16 in
    // `blob` (every path computes with the same values) and the HBM-bound
    // decode kernels read bf16 copies: fp32 tensor -> its bf16 bits
    bool bf16 = false;
    unsigned short* blob16 = nullptr;
    std::unordered_map<const float*, const unsigned short*> w16;
    // per layer, for each of the 4 matrices: {hi, lo, stored} descriptors of
    // W^T (128-row boxes); `stored` is W^T as fp32, or as bf16 for bf16
    // weights (the decode-batch GEMM reads it once and splits it on chip)
    std::vector<std::array<CUtensorMap, 12>> tc_maps;
    // the tied head: tok_emb [V][D] is already W^T of logits = x * tok_emb^T
    CUtensorMap tc_head_maps[3];
    float* tc_head_blob = nullptr;  // tok_emb hi, lo halves, then V zeros (the head has no bias)
};

struct fb2_model {
    fb2_model_desc desc{};
    int V = 0, ctx = 0, D = 0, L = 0, H = 0, hd = 0, F = 0;
    std::vector<DeviceModel> devs;
};

static std::vector<long long> param_numels(const fb2_model_desc& d) {
    long long D = d.d_model, F = 4LL * d.d_model;
    std::vector<long long> n;
    n.push_back((long long)d.vocab_size * D);
    n.push_back((long long)d.context_length * D);
    for (int l = 0; l < d.n_layers; l++) {
        long long b[12] = {D, D, D * 3 * D, 3 * D, D * D, D, D, D, D * F, F, F * D, D};
        n.insert(n.end(), b, b + 12);
    }
    n.push_back(D);
    n.push_back(D);
    return n;
}

// ---------------------------------------------------------------------------
// kernel launch configuration (per device, set once)
// ---------------------------------------------------------------------------
// Opts every kernel that takes dynamic shared memory into the device maximum
// (the opt-in limit covers static + dynamic shared memory of a block).
static void configure_kernels(int dev) {
    int optin = 0;
    CK(cudaDeviceGetAttribute(&optin, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev));
    auto setmax = [optin](const void* f, int) {
        cudaFuncAttributes a;
        CK(cudaFuncGetAttributes(&a, f));
        CK(cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, optin - (int)a.sharedSizeBytes));
    };
    setmax((const void*)k_gemv<1>, 227 * 1024);
    setmax((const void*)k_gemv<2>, 227 * 1024);
    setmax((const void*)k_gemv<4>, 227 * 1024);
    setmax((const void*)k_gemv<8>, 227 * 1024);
    setmax((const void*)k_gemv<16>, 227 * 1024);
    setmax((const void*)k_gemv<1, WBF16>, 227 * 1024);
    setmax((const void*)k_gemv<2, WBF16>, 227 * 1024);
    setmax((const void*)k_gemv<4, WBF16>, 227 * 1024);
    setmax((const void*)k_gemv<8, WBF16>, 227 * 1024);
    setmax((const void*)k_gemv<16, WBF16>, 227 * 1024);
    setmax((const void*)k_attn_prefill<4>, 227 * 1024);
    setmax((const void*)k_attn_prefill<8>, 227 * 1024);
    setmax((const void*)k_attn_prefill<16>, 227 * 1024);
    setmax((const void*)k_attn_prefill<32>, 227 * 1024);
    setmax((const void*)k_attn_prefill<64>, 227 * 1024);
    setmax((const void*)k_attn_prefill<128>, 227 * 1024);
    setmax((const void*)k_attn_prefill_rt<32>, 227 * 1024);
    setmax((const void*)k_attn_prefill_rt<64>, 227 * 1024);
    setmax((const void*)k_attn_prefill_rt<128>, 227 * 1024);
    setmax((const void*)k_attn_prefill_tc, 227 * 1024);
    setmax((const void*)k_head<1>, 227 * 1024);
    setmax((const void*)k_head<2>, 227 * 1024);
    setmax((const void*)k_head<4>, 227 * 1024);
    setmax((const void*)k_head<8>, 227 * 1024);
    setmax((const void*)k_head<16>, 227 * 1024);
    setmax((const void*)k_head<1, WBF16>, 227 * 1024);
    setmax((const void*)k_head<2, WBF16>, 227 * 1024);
    setmax((const void*)k_head<4, WBF16>, 227 * 1024);
    setmax((const void*)k_head<8, WBF16>, 227 * 1024);
    setmax((const void*)k_head<16, WBF16>, 227 * 1024);
    setmax((const void*)k_sample_step, 227 * 1024);
    setmax((const void*)k_gemm_tc<128>, 227 * 1024);
    setmax((const void*)k_gemm_tc_swab<64, false>, 227 * 1024);
    setmax((const void*)k_gemm_tc_swab<128, false>, 227 * 1024);
    setmax((const void*)k_gemm_tc_swab<64, true>, 227 * 1024);
    setmax((const void*)k_gemm_tc_swab<128, true>, 227 * 1024);
    setmax((const void*)k_sample_rows, 227 * 1024);
    setmax((const void*)k_decode_mega<1, false>, 0);
    setmax((const void*)k_decode_mega<2, false>, 0);
    setmax((const void*)k_decode_mega<4, false>, 0);
    setmax((const void*)k_decode_mega<8, false>, 0);
    setmax((const void*)k_decode_mega<1, true>, 0);
    setmax((const void*)k_decode_mega<2, true>, 0);
    setmax((const void*)k_decode_mega<4, true>, 0);
    setmax((const void*)k_decode_mega<8, true>, 0);
}

// ---------------------------------------------------------------------------
// persistent decode kernel: geometry and weight layout
// ---------------------------------------------------------------------------
static int mk_keys_per_chunk(int hd) { return MK_STAGE / (hd * 4); }
static int mk_maxc(int ctx, int hd) { return ceil_div(ctx, mk_keys_per_chunk(hd)); }
// Vocabulary entries per CTA slice, rounded up to a multiple of 4 so every
// shared-memory region after the slices stays 16-byte aligned.
static int mk_slice_max(int V, int nW) { return (ceil_div(V, nW) + 3) & ~3; }

// The persistent kernel's instantiation for MR rows and the layer path.
static const void* mk_kernel(int MR, bool hc) {
    if (hc)
        return MR == 1 ? (const void*)k_decode_mega<1, true>
             : MR == 2 ? (const void*)k_decode_mega<2, true>
             : MR == 4 ? (const void*)k_decode_mega<4, true>
                       : (const void*)k_decode_mega<8, true>;
    return MR == 1 ? (const void*)k_decode_mega<1, false>
         : MR == 2 ? (const void*)k_decode_mega<2, false>
         : MR == 4 ? (const void*)k_decode_mega<4, false>
                   : (const void*)k_decode_mega<8, false>;
}

// Dynamic shared memory of k_decode_mega<MR> with `nstage` ring stages
// (cs > 0: the head-cluster layout, clusters of cs CTAs).
static size_t mk_smem(const fb2_model& m, int MR, int nW, int nstage, int cs = 0, int sb = MK_STAGE) {
    return (size_t)nstage * sb +
           mk_aux_bytes(MR, m.D, m.F, m.H, m.ctx, mk_slice_max(m.V, nW), mk_maxc(m.ctx, m.hd), nstage) +
           (cs > 0 ? mk_hc_bytes(MR, m.D, m.F, m.hd, m.ctx, cs, nW, m.L) : 0) + 256;
}

// Ring stages that fit next to the kernel's other shared memory (0: does not fit).
static int mk_nstage(const fb2_model& m, int MR, int nW, int device, int cs = 0, int sb = MK_STAGE) {
    int optin = 0;
    CK(cudaDeviceGetAttribute(&optin, cudaDevAttrMaxSharedMemoryPerBlockOptin, device));
    cudaFuncAttributes fa;
    const void* f = mk_kernel(MR, cs > 0);
    CK(cudaFuncGetAttributes(&fa, f));
    const long long avail = (long long)optin - (long long)fa.sharedSizeBytes;
    int ns = 16;
    while (ns >= 4 && (long long)mk_smem(m, MR, nW, ns, cs, sb) > avail) ns--;
    return ns >= 4 ? ns : 0;
}

// Clusters of `cs` CTAs of k_decode_mega<1> that can be resident at once.
static int mk_max_clusters(const fb2_model& m, int nW, int cs, int device) {
    const int ns = mk_nstage(m, 1, nW, device, cs);
    if (ns == 0) return 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(nW);
    cfg.blockDim = dim3(MK_THREADS);
    cfg.dynamicSmemBytes = mk_smem(m, 1, nW, ns, cs);
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = cs;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, mk_kernel(1, true), &cfg) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    return n;
}

// ---- bf16 weights ---------------------------------------------------------------
// Round to the nearest bf16 value (ties to even), kept as fp32.
static float bf16_round_host(float x) {
    uint32_t u;
    std::memcpy(&u, &x, 4);
    if ((u & 0x7F800000u) != 0x7F800000u) u = (u + 0x7FFFu + ((u >> 16) & 1u)) & 0xFFFF0000u;
    float r;
    std::memcpy(&r, &u, 4);
    return r;
}
// bf16 bits of values that are already bf16-representable fp32.
__global__ void k_to_bf16_bits(const float* __restrict__ x, long long n, unsigned short* __restrict__ y) {
    pdl_wait();
    for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x)
        y[i] = (unsigned short)(__float_as_uint(x[i]) >> 16);
}

// ---- tensor-core GEMM support ----------------------------------------------
static PFN_cuTensorMapEncodeTiled_v12000 tc_encode_fn() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q{};
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
    });
    return fn;
}
// 2-D fp32 row-major [outer][inner] map, 128-byte swizzled boxes of
// 32 x box_outer elements.
static bool tc_encode(CUtensorMap* map, const float* base, uint64_t inner, uint64_t outer, uint32_t box_outer) {
    auto fn = tc_encode_fn();
    if (!fn) return false;
    const cuuint64_t dims[2] = {inner, outer};
    const cuuint64_t strides[1] = {inner * 4};
    const cuuint32_t box[2] = {32, box_outer};
    const cuuint32_t estr[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, const_cast<float*>(base), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
static void launch_split_tf32(cudaStream_t st, const float* x, size_t n, float* hi, float* lo) {
    const size_t n4 = n / 4;
    const int blocks = (int)std::min<size_t>(4096, (n4 + 255) / 256);
    launch_pdl(k_split_tf32, std::max(blocks, 1), 256, 0, st, reinterpret_cast<const float4*>(x), n4,
                                                      reinterpret_cast<float4*>(hi), reinterpret_cast<float4*>(lo));
}
static void launch_split_tf32_transpose(cudaStream_t st, const float* W, int K, int N, float* hiT, float* loT,
                                        float* rawT = nullptr) {
    launch_pdl(k_split_tf32_transpose, dim3(ceil_div(N, 32), ceil_div(K, 32)), dim3(32, 8), 0, st, W, K, N, hiT, loT,
               rawT);
}
// 2-D bf16 row-major [outer][inner] map, unswizzled boxes of 32 x box_outer
// elements (64-byte rows).
static bool tc_encode_bf16(CUtensorMap* map, const unsigned short* base, uint64_t inner, uint64_t outer,
                           uint32_t box_outer) {
    auto fn = tc_encode_fn();
    if (!fn) return false;
    const cuuint64_t dims[2] = {inner, outer};
    const cuuint64_t strides[1] = {inner * 2};
    const cuuint32_t box[2] = {32, box_outer};
    const cuuint32_t estr[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<unsigned short*>(base), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// TF32 hi/lo copies of every projection, transposed to W^T [N][K], W^T as
// stored (fp32, or the bf16 bits of bf16 weights, whose TF32 hi half is the
// value itself), and their descriptors (boxes of 32 K x 128 N rows).
// FORGE_B200_GEMM=simt leaves the tensor-core path off.
static void tc_setup(const fb2_model& m, DeviceModel& dm) {
    dm.tc_ok = false;
    const char* env = getenv("FORGE_B200_GEMM");
    if (env && std::string(env) == "simt") return;
    if (!tc_encode_fn() || (m.D % 32) != 0) return;
    const size_t D = m.D, F = m.F;
    const size_t per_layer = 3 * D * D + D * D + D * F + F * D;
    dm.tc_blob = dalloc<float>(3 * per_layer * m.L);
    dm.tc_maps.resize(m.L);
    for (int l = 0; l < m.L; l++) {
        const LayerW& w = dm.layers[l];
        const float* src[4] = {w.qkv_w, w.proj_w, w.fc_w, w.mproj_w};
        const size_t Ks[4] = {D, D, D, F}, Ns[4] = {3 * D, D, F, D};
        float* at = dm.tc_blob + 3 * per_layer * l;
        for (int j = 0; j < 4; j++) {
            const size_t n = Ks[j] * Ns[j];
            float* hi = at;
            float* lo = at + n;
            float* raw = at + 2 * n;
            CUtensorMap* mp = &dm.tc_maps[l][3 * j];
            launch_split_tf32_transpose(0, src[j], (int)Ks[j], (int)Ns[j], hi, lo, dm.bf16 ? nullptr : raw);
            if (!tc_encode(&mp[0], hi, Ks[j], Ns[j], 128) || !tc_encode(&mp[1], lo, Ks[j], Ns[j], 128)) return;
            if (dm.bf16) {
                unsigned short* raw16 = reinterpret_cast<unsigned short*>(raw);
                k_to_bf16_bits<<<(int)std::min<size_t>(4096, (n + 255) / 256), 256>>>(hi, (long long)n, raw16);
                if (!tc_encode_bf16(&mp[2], raw16, Ks[j], Ns[j], 128)) return;
            } else if (!tc_encode(&mp[2], raw, Ks[j], Ns[j], 128)) {
                return;
            }
            at += 3 * n;
        }
    }
    {
        const size_t nv = (size_t)m.V * D;
        dm.tc_head_blob = dalloc<float>(2 * nv + (size_t)m.V);
        launch_split_tf32(0, dm.tok_emb, nv, dm.tc_head_blob, dm.tc_head_blob + nv);
        CK(cudaMemset(dm.tc_head_blob + 2 * nv, 0, (size_t)m.V * 4));
        if (!tc_encode(&dm.tc_head_maps[0], dm.tc_head_blob, D, m.V, 128) ||
            !tc_encode(&dm.tc_head_maps[1], dm.tc_head_blob + nv, D, m.V, 128))
            return;
        if (dm.bf16) {
            auto it = dm.w16.find(dm.tok_emb);
            if (it == dm.w16.end() || !tc_encode_bf16(&dm.tc_head_maps[2], it->second, D, m.V, 128)) return;
        } else if (!tc_encode(&dm.tc_head_maps[2], dm.tok_emb, D, m.V, 128)) {
            return;
        }
    }
    CK(cudaDeviceSynchronize());
    dm.tc_ok = true;
    const char* aenv = getenv("FORGE_B200_ATTN");
    dm.attn_tc = m.hd == ATC_HD && !(aenv && std::string(aenv) == "simt");
}

// Re-lays every projection W[K][N] as consecutive column strips [K][w_c],
// one per CTA (the split k_decode_mega streams), and uploads the layer table.
// Head-cluster geometry for this model on this device, if it applies:
// clusters of 4 CTAs, one per head; at least half as many MLP CTAs as
// attention CTAs; every slice no wider than the column kernels take.
static bool mk_hc_plan(const fb2_model& m, DeviceModel& dm) {
    const char* env = getenv("FORGE_B200_MK");
    if (env && std::string(env) == "strips") return false;
    const char* ecs = getenv("FORGE_B200_MK_CS");
    const int want = ecs ? atoi(ecs) : 0;
    // clusters of 8 when 8 CTAs per head fit the resident grid, else of 4
    for (int cs : {8, 4}) {
        if (want && cs != want) continue;
        if (m.hd % cs != 0 || m.D % (4 * cs) != 0 || m.D > 1024 || 3 * m.hd / cs > 256) continue;
        const int nhead = m.H * cs;
        int nW = (dm.sm_count / cs) * cs;
        const int nc = mk_max_clusters(m, nW, cs, dm.device);
        nW = std::min(nW, nc * cs);
        if (nhead > nW || ceil_div(m.F, nW) > 256 || nW < 32) continue;
        if (mk_slice_max(m.V, nW) > MK_SLICE_MAX) continue;
        dm.mk_hc = true;
        dm.mk_cs = cs;
        dm.mk_nhead = nhead;
        dm.mk_nW = nW;
        return true;
    }
    return false;
}

static void mk_setup(const fb2_model& m, DeviceModel& dm, const float* const* params) {
    dm.mk_ok = false;
    dm.mk_hc = false;
    int nW = dm.sm_count;
    if (!(m.hd == 32 || m.hd == 64)) return;
    if (mk_maxc(m.ctx, m.hd) > 32) return;
    if (m.V <= m.ctx) return;  // the ban of a whole window could then cover the vocabulary
    if (mk_slice_max(m.V, nW) > MK_SLICE_MAX || nW > 256) return;
    if (m.D * 4 > MK_STAGE) return;
    if (8 * ceil_div(4 * m.D, nW) > 512) return;  // strip outputs staged in a 512-float scratch
    if (mk_nstage(m, 1, nW, dm.device) == 0) return;
    const bool hc = mk_hc_plan(m, dm);
    if (hc) nW = dm.mk_nW;
    const size_t D = m.D, F = m.F;
    const size_t per_layer = 3 * D * D + D * D + D * F + F * D;
    dm.relaid = dalloc<float>(per_layer * m.L);
    if (hc) dm.mk_fold = dalloc<float>((size_t)m.L * 2 * (3 * D + F));
    std::vector<float> tmp(std::max(3 * D * D, D * F));
    std::vector<MkLayer> host(m.L);
    for (int l = 0; l < m.L; l++) {
        const float* const* q = params + 2 + 12 * l;
        struct { const float* W; size_t K, N; } mats[4] = {{q[2], D, 3 * D}, {q[4], D, D}, {q[8], D, F}, {q[10], F, D}};
        size_t off = per_layer * l;
        for (int ph = 0; ph < 4; ph++) {
            const size_t K = mats[ph].K, N = mats[ph].N;
            const float* W = mats[ph].W;
            if (hc) {
                // head CTA c = (head h, rank r) reads QKV as [D][3 hq] (its q, k, v
                // columns of head h) and proj as [hd][D/cs] (head h's rows, its
                // column quarter); MLP CTA j reads fc as [D][J_j] (its hidden
                // units); mlp.proj keeps its layout (rows j0..j1 are contiguous)
                const size_t cs = dm.mk_cs, hd = m.hd, hq = hd / cs, nhead = dm.mk_nhead, nmlp = nW;
                size_t o = 0;
                if (ph == MK_QKV) {
                    // LN1's gains folded into the weights: g_k W[k][c]
                    const float* g = q[0];
                    for (size_t c = 0; c < nhead; c++) {
                        const size_t h = c / cs, r = c % cs;
                        for (size_t k = 0; k < K; k++)
                            for (size_t part = 0; part < 3; part++)
                                for (size_t i = 0; i < hq; i++)
                                    tmp[o + k * 3 * hq + part * hq + i] = g[k] * W[k * N + part * D + h * hd + r * hq + i];
                        o += K * 3 * hq;
                    }
                } else if (ph == MK_PROJ) {
                    const size_t wp = D / cs;
                    for (size_t c = 0; c < nhead; c++) {
                        const size_t h = c / cs, r = c % cs;
                        for (size_t d = 0; d < hd; d++)
                            std::memcpy(&tmp[o + d * wp], W + (h * hd + d) * N + r * wp, wp * sizeof(float));
                        o += hd * wp;
                    }
                } else if (ph == MK_FC) {
                    // LN2's gains folded into the weights
                    const float* g = q[6];
                    for (size_t j = 0; j < nmlp; j++) {
                        const size_t j0 = 4 * (j * (F / 4) / nmlp), j1 = 4 * ((j + 1) * (F / 4) / nmlp), w = j1 - j0;
                        for (size_t k = 0; k < K; k++)
                            for (size_t i = 0; i < w; i++) tmp[K * j0 + k * w + i] = g[k] * W[k * N + j0 + i];
                    }
                } else {
                    std::memcpy(tmp.data(), W, K * N * sizeof(float));
                }
            } else {
                for (int c = 0; c < nW; c++) {
                    const size_t n0 = (size_t)c * N / nW, n1 = (size_t)(c + 1) * N / nW, w = n1 - n0;
                    for (size_t k = 0; k < K; k++)
                        std::memcpy(&tmp[K * n0 + k * w], W + k * N + n0, w * sizeof(float));
                }
            }
            CK(cudaMemcpy(dm.relaid + off, tmp.data(), K * N * sizeof(float), cudaMemcpyHostToDevice));
            host[l].w[ph] = dm.relaid + off;
            off += K * N;
        }
        if (hc) {
            // per qkv / fc column: (S, B) of the folded LayerNorm, in double:
            // S_c = sum_k (g_k W[k][c]) as the kernel multiplies, B_c = sum_k beta_k W[k][c] + bias_c
            std::vector<float> fold(2 * (3 * D + F));
            auto fold_cols = [&](const float* W, size_t N, const float* g, const float* beta, const float* bias,
                                 float* out) {
                std::vector<double> sS(N, 0.0), sB(N, 0.0);
                for (size_t k = 0; k < D; k++)
                    for (size_t c = 0; c < N; c++) {
                        sS[c] += (double)(g[k] * W[k * N + c]);
                        sB[c] += (double)beta[k] * (double)W[k * N + c];
                    }
                for (size_t c = 0; c < N; c++) {
                    out[2 * c] = (float)sS[c];
                    out[2 * c + 1] = (float)(sB[c] + (double)bias[c]);
                }
            };
            fold_cols(q[2], 3 * D, q[0], q[1], q[3], fold.data());
            fold_cols(q[8], F, q[6], q[7], q[9], fold.data() + 2 * 3 * D);
            CK(cudaMemcpy(dm.mk_fold + (size_t)l * fold.size(), fold.data(), fold.size() * sizeof(float),
                          cudaMemcpyHostToDevice));
            host[l].fold[0] = dm.mk_fold + (size_t)l * fold.size();
            host[l].fold[1] = host[l].fold[0] + 2 * 3 * D;
        }
        const LayerW& lw = dm.layers[l];
        host[l].b[MK_QKV] = lw.qkv_b;
        host[l].b[MK_PROJ] = lw.proj_b;
        host[l].b[MK_FC] = lw.fc_b;
        host[l].b[MK_PROJ2] = lw.mproj_b;
        host[l].ln1w = lw.ln1_w;
        host[l].ln1b = lw.ln1_b;
        host[l].ln2w = lw.ln2_w;
        host[l].ln2b = lw.ln2_b;
    }
    dm.d_mk_layers = dalloc<MkLayer>(m.L);
    CK(cudaMemcpy(dm.d_mk_layers, host.data(), m.L * sizeof(MkLayer), cudaMemcpyHostToDevice));
    dm.mk_nW = nW;
    dm.mk_ok = true;
}

// ---------------------------------------------------------------------------
// session
// ---------------------------------------------------------------------------
struct ChunkPlan {
    int row_off;      // first entry in the row table
    int rows;         // rows in this chunk
    int qblk_off, nqblk;    // query blocks of <= 64 rows (SIMT attention)
    int qblk2_off, nqblk2;  // query blocks of <= 128 rows (tensor-core attention)
    int slot_off, nslots;  // entries in last_row / out_slot tables
};

struct DeviceSession {
    fb2_model* model = nullptr;
    const DeviceModel* dm = nullptr;
    int device = 0;
    int slot0 = 0, nslots = 0;  // global slot range
    cudaStream_t own_stream = nullptr, stream = nullptr;

    // per-slot state
    int *d_len = nullptr, *d_count = nullptr, *d_done = nullptr, *d_hist = nullptr;
    // tokens whose K/V the slot's cache holds at positions 0.. (the window of
    // the last host-path generate, when it never slid); empty = unknown.  A
    // later generate whose prompt starts with them prefills only the rest
    // (a chat turn resubmits the whole history, Program.cs:736-765).
    std::vector<std::vector<int>> kv_tokens;
    int hist_cap = 0;
    float* d_kv = nullptr;
    long long kv_slot_stride = 0, kv_layer_stride = 0, v_offset = 0;

    // rows
    int row_cap = 0;
    int *d_row_seq = nullptr, *d_row_pos = nullptr, *d_row_hidx = nullptr, *d_row_active = nullptr;
    int* d_ones = nullptr;
    float *d_x = nullptr, *d_x2 = nullptr, *d_ln = nullptr, *d_q = nullptr, *d_att = nullptr, *d_h = nullptr;
    float *d_ahi = nullptr, *d_alo = nullptr;  // TF32 halves of a GEMM's A operand
    int* d_tc_err = nullptr;
    float *d_ahi2 = nullptr, *d_alo2 = nullptr;  // TF32 halves of the MLP hidden rows (prefill)
    float* d_tc_part = nullptr;  // split-K partial tiles of the decode GEMM
    size_t tc_part_cap = 0;
    float *d_logits = nullptr, *d_lnf = nullptr;
    float* d_attn_part = nullptr;
    int attn_nsplit = 0;
    float* d_gemv_part = nullptr;
    size_t gemv_part_cap = 0;
    unsigned int* d_tickets = nullptr;

    // call tables (uploaded once per call)
    int* d_tab = nullptr;
    size_t tab_cap = 0;  // ints
    int* h_tab = nullptr;  // pinned staging
    size_t h_tab_cap = 0;
    cudaEvent_t tab_event = nullptr;
    bool tab_event_pending = false;
    double* d_uni = nullptr;
    size_t uni_cap = 0;
    int* d_out = nullptr;
    size_t out_cap = 0;

    // decode graph
    cudaGraphExec_t graph = nullptr;
    int graph_n = -1;
    long long graph_kernels = 0;  // kernel nodes in the captured step
    cudaStream_t graph_stream = nullptr;

    std::vector<DotNetRandom> rngs;  // FB2_RNG_SESSION streams of this device's slots

    // persistent decode kernel (k_decode_mega) state
    bool mk_use = false;
    unsigned long long *mk_xq = nullptr, *mk_xkv = nullptr, *mk_xx2 = nullptr, *mk_xh = nullptr, *mk_xx = nullptr;
    unsigned long long *mk_xpart = nullptr, *mk_hdr = nullptr;
    float *mk_xacc = nullptr, *mk_cval = nullptr;
    int* mk_cidx = nullptr;
    unsigned int* mk_stepdone = nullptr;
    int *mk_err = nullptr, *mk_rows = nullptr;
    unsigned int mk_gstep = 0;
    size_t mk_tagged_words = 0;
    unsigned long long* mk_acc = nullptr;  // head-cluster layout: counted fixed-point accumulators
    size_t mk_acc_words = 0;
    unsigned long long* mk_trace = nullptr;
    int mk_trace_steps = 0;

    // stats
    fb2_stats_t stats{};
    cudaEvent_t ev0 = nullptr, ev1 = nullptr;
    // test hook (fb2_test_mk_withhold): the next persistent launch withholds
    // one CTA's q words and waits at most test_wait_ns
    int test_withhold_cta = -1;
    unsigned long long test_wait_ns = 0;
};

struct fb2_session {
    fb2_model* model = nullptr;
    int max_seqs = 0;
    std::vector<DeviceSession*> ds;
    fb2_uniform_cb ucb = nullptr;  // FB2_RNG_CALLBACK source
    void* ucb_user = nullptr;
};

// Zeroes the persistent kernel's tagged words, counters and error flag and
// restarts its step numbering (tags compare against 1 + step * (L+1) + layer,
// so zeroed words never match).
static void mk_reset(DeviceSession& s) {
    CK(cudaMemsetAsync(s.mk_xq, 0, s.mk_tagged_words * 8, s.stream));
    CK(cudaMemsetAsync(s.mk_stepdone, 0, sizeof(unsigned int), s.stream));
    CK(cudaMemsetAsync(s.mk_err, 0, sizeof(int), s.stream));
    if (s.mk_acc) CK(cudaMemsetAsync(s.mk_acc, 0, s.mk_acc_words * 8, s.stream));
    s.mk_gstep = 0;
}

// Buffers of k_decode_mega for up to MK_MAX_ROWS rows on this device.
// FORGE_B200_DECODE=graph keeps the multi-kernel graph path instead.
static void mk_session_alloc(DeviceSession& s) {
    const fb2_model& m = *s.model;
    const DeviceModel& dm = *s.dm;
    const char* env = getenv("FORGE_B200_DECODE");
    s.mk_use = dm.mk_ok && !(env && std::string(env) == "graph");
    if (!s.mk_use) return;
    const size_t R = MK_MAX_ROWS, D = m.D, F = m.F, nW = dm.mk_nW;
    const size_t units = R * m.H * mk_maxc(m.ctx, m.hd);
    s.mk_tagged_words = R * D + R * 2 * D + R * D + R * F + R * D + units * (m.hd + 2) + R * nW * 9;
    s.mk_xq = dalloc<unsigned long long>(s.mk_tagged_words);
    s.mk_xkv = s.mk_xq + R * D;
    s.mk_xx2 = s.mk_xkv + R * 2 * D;
    s.mk_xh = s.mk_xx2 + R * D;
    s.mk_xx = s.mk_xh + R * F;
    s.mk_xpart = s.mk_xx + R * D;
    s.mk_hdr = s.mk_xpart + units * (m.hd + 2);
    s.mk_xacc = dalloc<float>(units * m.hd);
    const size_t slice = mk_slice_max(m.V, (int)nW);
    s.mk_cval = dalloc<float>(R * nW * slice);
    s.mk_cidx = dalloc<int>(R * nW * slice);
    s.mk_stepdone = dalloc<unsigned int>(1);
    s.mk_err = dalloc<int>(1);
    if (dm.mk_hc) {
        s.mk_acc_words = 2 * (size_t)m.L * 2 * MK_MAX_ROWS * D;
        s.mk_acc = dalloc<unsigned long long>(s.mk_acc_words);
    }
    s.mk_rows = dalloc<int>(R);
    if (const char* tr = getenv("FORGE_B200_MK_TRACE")) {  // per-phase timestamps of the first steps
        s.mk_trace_steps = std::max(0, std::min(64, atoi(tr)));
        if (s.mk_trace_steps > 0) {
            s.mk_trace = dalloc<unsigned long long>((size_t)nW * s.mk_trace_steps * MK_TRACE_POINTS);
            CK(cudaMemset(s.mk_trace, 0, (size_t)nW * s.mk_trace_steps * MK_TRACE_POINTS * 8));
        }
    }
    std::vector<int> rows(R);
    for (size_t i = 0; i < R; i++) rows[i] = (int)std::min(i, (size_t)std::max(s.nslots - 1, 0));
    CK(cudaMemcpy(s.mk_rows, rows.data(), R * sizeof(int), cudaMemcpyHostToDevice));
    mk_reset(s);
    CK(cudaStreamSynchronize(s.stream));
}

static void session_free(DeviceSession* s) {
    if (!s) return;
    cudaSetDevice(s->device);
    if (s->graph) cudaGraphExecDestroy(s->graph);
    dfree(s->d_len); dfree(s->d_count); dfree(s->d_done); dfree(s->d_hist); dfree(s->d_kv);
    dfree(s->d_row_seq); dfree(s->d_row_pos); dfree(s->d_row_hidx); dfree(s->d_row_active); dfree(s->d_ones);
    dfree(s->d_x); dfree(s->d_x2); dfree(s->d_ln); dfree(s->d_q); dfree(s->d_att); dfree(s->d_h);
    dfree(s->d_ahi); dfree(s->d_alo); dfree(s->d_ahi2); dfree(s->d_alo2); dfree(s->d_tc_err); dfree(s->d_tc_part);
    dfree(s->d_logits); dfree(s->d_lnf); dfree(s->d_attn_part); dfree(s->d_gemv_part); dfree(s->d_tickets);
    dfree(s->d_tab); dfree(s->d_uni); dfree(s->d_out);
    dfree(s->mk_xq); dfree(s->mk_xacc); dfree(s->mk_cval); dfree(s->mk_cidx); dfree(s->mk_stepdone);
    dfree(s->mk_err); dfree(s->mk_rows); dfree(s->mk_trace); dfree(s->mk_acc);
    if (s->h_tab) cudaFreeHost(s->h_tab);
    if (s->tab_event) cudaEventDestroy(s->tab_event);
    if (s->ev0) cudaEventDestroy(s->ev0);
    if (s->ev1) cudaEventDestroy(s->ev1);
    if (s->own_stream) cudaStreamDestroy(s->own_stream);
    delete s;
}

// ---------------------------------------------------------------------------
// launch helpers
// ---------------------------------------------------------------------------
static void launch_layernorm(DeviceSession& s, int rows, const float* x, const float* w, const float* b, float* y,
                             const int* row_map, float* y_lo = nullptr) {
    int D = s.model->D;
    int per = ceil_div(D, 32);
    dim3 grid(ceil_div(rows, 8)), block(256);
#define LN_CASE(P) \
    if (per <= P) { s.stats.kernel_launches++; launch_pdl(k_layernorm<P>, grid, block, 0, s.stream, rows, D, x, w, b, y, row_map, y_lo); return; }
    LN_CASE(1) LN_CASE(2) LN_CASE(4) LN_CASE(8) LN_CASE(16) LN_CASE(24) LN_CASE(32) LN_CASE(48) LN_CASE(64)
#undef LN_CASE
    fail(FB2_UNSUPPORTED, "d_model too large for the LayerNorm kernel");
}

// Split-K geometry of k_gemv for a [K][N] weight: S k-splits of kchunk rows.
struct GemvSplit {
    int S, kchunk;
};
static GemvSplit gemv_split(int sm_count, int K, int N) {
    int nblk = ceil_div(N, 64);
    int target = 2 * sm_count;
    int S = std::max(1, ceil_div(target, nblk));
    S = std::min(S, std::max(1, K / 16));
    int kchunk = ceil_div(ceil_div(K, S), 16) * 16;
    if (kchunk > kGemvMaxKChunk) kchunk = kGemvMaxKChunk;
    return GemvSplit{ceil_div(K, kchunk), kchunk};
}

template <int MR>
static void launch_gemv_mr(DeviceSession& s, int M, int K, int N, const float* A, const float* W, const Epi& e) {
    int nblk = ceil_div(N, 64);
    const GemvSplit sp = gemv_split(s.dm->sm_count, K, N);
    const int S = sp.S, kchunk = sp.kchunk;
    size_t need = (size_t)S * M * N;
    if (S > 1 && need > s.gemv_part_cap) fail(FB2_UNSUPPORTED, "split-K scratch too small");
    size_t smem = (size_t)MR * kchunk * 4 + (size_t)16 * MR * 64 * 4;
    s.stats.kernel_launches++;
    auto it = s.dm->w16.find(W);
    if (it != s.dm->w16.end())
        launch_pdl(k_gemv<MR, WBF16>, dim3(nblk, S), 256, smem, s.stream, M, K, N, kchunk, A, it->second, s.d_gemv_part,
                                                                  s.d_tickets, e);
    else
        launch_pdl(k_gemv<MR>, dim3(nblk, S), 256, smem, s.stream, M, K, N, kchunk, A, W, s.d_gemv_part, s.d_tickets, e);
}

// y = A * W (+ epilogue) for M rows.
static void launch_linear(DeviceSession& s, int M, int K, int N, const float* A, const float* W, Epi e);

// Tensor-core (3xTF32) GEMM: from kTcMinRows rows, 128 x 128 output tiles;
// decode batches of kMaxGemvRows+1 .. kTcMinRows-1 rows use the swapped
// operands (weights as the 128-row side, read once) with split-K.
constexpr int kTcMinRows = 512;

// The launch of one tensor-core projection; false when it does not apply.
// a_split: A's TF32 halves are already in ahi / alo (written by the producer
// of A); prefill only.
// bmaps: {hi, lo, stored} descriptors of W^T; w_bf16: `stored` is bf16.
static bool launch_gemm_tc(cudaStream_t st, int sm_count, int M, int K, int N, const float* A, float* ahi, float* alo,
                           const CUtensorMap* bmaps, Epi e, int* err, float* part, size_t part_cap, int64_t* launches,
                           bool w_bf16, bool a_split = false) {
    if (M <= kMaxGemvRows || (K % 4) || (N % 4)) return false;
    TcMaps maps;
    maps.b_hi = bmaps[0];
    maps.b_lo = bmaps[1];
    if (M >= kTcMinRows) {
        if (!a_split) {
            launch_split_tf32(st, A, (size_t)M * K, ahi, alo);
            (*launches)++;
        }
        if (!tc_encode(&maps.a_hi, ahi, K, M, TC_BM) || !tc_encode(&maps.a_lo, alo, K, M, TC_BM))
            fail(FB2_CUDA_ERROR, "cuTensorMapEncodeTiled failed for a GEMM operand");
        (*launches)++;
        const int tiles = ceil_div(N, 128) * ceil_div(M, TC_BM);
        launch_pdl(k_gemm_tc<128>, std::min(tiles, sm_count), TCP_THREADS, TcCfg<128>::SMEM, st, maps, M, N, K, e, err);
        return true;
    }
    // decode batches: the kernel splits A's tiles and W^T's stored tiles
    // itself (maps.a_hi = A, maps.b_hi = W^T as stored)
    const int bnb = M <= 64 ? 64 : 128;
    if (!tc_encode(&maps.a_hi, A, K, M, bnb)) fail(FB2_CUDA_ERROR, "cuTensorMapEncodeTiled failed for a GEMM operand");
    maps.a_lo = maps.a_hi;
    maps.b_hi = bmaps[2];
    maps.b_lo = bmaps[2];
    const int tiles = ceil_div(N, 128) * ceil_div(M, bnb), nk = ceil_div(K, TC_BK);
    int S = std::max(1, std::min({kTcSplitMax, nk, sm_count / tiles}));
    S = ceil_div(nk, ceil_div(nk, S));  // balanced k blocks per split
    if ((size_t)S * M * N > part_cap) S = 1;
    dim3 grid(ceil_div(N, 128), ceil_div(M, bnb), S);
    (*launches)++;
    if (bnb == 64) {
        if (w_bf16) launch_pdl(k_gemm_tc_swab<64, true>, grid, TCS_THREADS, TcSwabCfg<64>::SMEM, st, maps, M, N, K, e, err, part);
        else launch_pdl(k_gemm_tc_swab<64, false>, grid, TCS_THREADS, TcSwabCfg<64>::SMEM, st, maps, M, N, K, e, err, part);
    } else {
        if (w_bf16) launch_pdl(k_gemm_tc_swab<128, true>, grid, TCS_THREADS, TcSwabCfg<128>::SMEM, st, maps, M, N, K, e, err, part);
        else launch_pdl(k_gemm_tc_swab<128, false>, grid, TCS_THREADS, TcSwabCfg<128>::SMEM, st, maps, M, N, K, e, err, part);
    }
    if (S > 1) {
        const size_t n4 = (size_t)M * N / 4;
        (*launches)++;
        launch_pdl(k_splitk_reduce, (int)std::min<size_t>((n4 + 255) / 256, 4 * (size_t)sm_count), 256, 0, st, part, S, M, N, e);
    }
    return true;
}

// y = A * W (+ epilogue) for M rows.  `bmaps` (TF32 hi/lo descriptors of W)
// selects the tensor-core GEMM when it applies.
static void launch_linear(DeviceSession& s, int M, int K, int N, const float* A, const float* W, Epi e,
                          const CUtensorMap* bmaps) {
    // bf16 weights: batches of <= 16 rows stay on the bf16 gemv (half the
    // bytes); larger batches take the tensor cores like fp32 weights (the
    // TF32 halves of the bf16-rounded values are exact), which measured
    // faster than a bf16 gemv pass per 16 rows
    if (bmaps && s.d_ahi && !(s.dm->bf16 && M <= kMaxGemvRows) &&
        launch_gemm_tc(s.stream, s.dm->sm_count, M, K, N, A, s.d_ahi, s.d_alo, bmaps, e, s.d_tc_err, s.d_tc_part,
                       s.tc_part_cap, &s.stats.kernel_launches, s.dm->bf16))
        return;
    launch_linear(s, M, K, N, A, W, e);
}

// Prefill projection whose operand's TF32 halves the producer already wrote
// (ahi / alo); the caller checked that the tensor-core path applies.
static void launch_linear_split(DeviceSession& s, int M, int K, int N, float* ahi, float* alo, const CUtensorMap* bmaps,
                                Epi e) {
    if (!launch_gemm_tc(s.stream, s.dm->sm_count, M, K, N, nullptr, ahi, alo, bmaps, e, s.d_tc_err, s.d_tc_part,
                        s.tc_part_cap, &s.stats.kernel_launches, s.dm->bf16, true))
        fail(FB2_CUDA_ERROR, "tensor-core GEMM refused a pre-split operand");
}

static void launch_linear(DeviceSession& s, int M, int K, int N, const float* A, const float* W, Epi e) {
    if (M <= kMaxGemvRows) {
        if (M <= 1) launch_gemv_mr<1>(s, M, K, N, A, W, e);
        else if (M <= 2) launch_gemv_mr<2>(s, M, K, N, A, W, e);
        else if (M <= 4) launch_gemv_mr<4>(s, M, K, N, A, W, e);
        else if (M <= 8) launch_gemv_mr<8>(s, M, K, N, A, W, e);
        else launch_gemv_mr<16>(s, M, K, N, A, W, e);
        return;
    }
    if (M <= 64) {
        // decode batches of up to 64 rows: stream W once per 16 rows
        for (int m0 = 0; m0 < M; m0 += kMaxGemvRows) {
            int mm = std::min(kMaxGemvRows, M - m0);
            Epi e2 = e;
            const float* A2 = A + (size_t)m0 * K;
            if (e.kind == EPI_QKV) {
                e2.out = e.out + (size_t)m0 * e.D;
                e2.R.seq = e.R.seq + m0; e2.R.pos = e.R.pos + m0; e2.R.active = e.R.active + m0;
                if (e.R.hidx) e2.R.hidx = e.R.hidx + m0;
            } else {
                e2.out = e.out + (size_t)m0 * N;
                if (e.resid) e2.resid = e.resid + (size_t)m0 * N;
            }
            if (mm <= 8) launch_gemv_mr<8>(s, mm, K, N, A2, W, e2);
            else launch_gemv_mr<16>(s, mm, K, N, A2, W, e2);
        }
        return;
    }
    if (M <= 1024) {
        dim3 grid(ceil_div(N, 128), ceil_div(M, 64));
        s.stats.kernel_launches++; launch_pdl(k_gemm_tiled<64>, grid, 256, 0, s.stream, M, K, N, A, W, e);
    } else {
        dim3 grid(ceil_div(N, 128), ceil_div(M, 128));
        s.stats.kernel_launches++; launch_pdl(k_gemm_tiled<128>, grid, 256, 0, s.stream, M, K, N, A, W, e);
    }
}

static Epi make_epi(int kind, const float* bias, const float* resid, float* out) {
    Epi e{};
    e.kind = kind;
    e.bias = bias;
    e.resid = resid;
    e.out = out;
    return e;
}

template <int HD>
static void launch_attn_decode_hd(DeviceSession& s, int M, int layer, Rows R) {
    const fb2_model& m = *s.model;
    float scale = 1.0f / sqrtf((float)m.hd);  // Layers.cs:174
    const float* kvl = s.d_kv + (size_t)layer * s.kv_layer_stride;
    s.stats.kernel_launches++; launch_pdl(k_attn_decode_partial<HD>, dim3(M, m.H, s.attn_nsplit), 128, 0, s.stream, 
        s.d_q, kvl, s.kv_slot_stride, s.v_offset, m.H, m.ctx, scale, R, s.d_attn_part, s.attn_nsplit);
    s.stats.kernel_launches++; launch_pdl(k_attn_decode_combine<HD>, dim3(M, m.H), 64, 0, s.stream, s.d_attn_part, m.H, s.attn_nsplit, R, s.d_att);
}

static void launch_attn_decode(DeviceSession& s, int M, int layer, Rows R) {
    switch (s.model->hd) {
    case 4: launch_attn_decode_hd<4>(s, M, layer, R); break;
    case 8: launch_attn_decode_hd<8>(s, M, layer, R); break;
    case 16: launch_attn_decode_hd<16>(s, M, layer, R); break;
    case 32: launch_attn_decode_hd<32>(s, M, layer, R); break;
    case 64: launch_attn_decode_hd<64>(s, M, layer, R); break;
    case 128: launch_attn_decode_hd<128>(s, M, layer, R); break;
    default: fail(FB2_UNSUPPORTED, "head_dim must be a power of two in [4, 128]");
    }
}

template <int HD>
static void launch_attn_prefill_hd(DeviceSession& s, int nblk, const int4* qblk, int layer) {
    const fb2_model& m = *s.model;
    float scale = 1.0f / sqrtf((float)m.hd);
    const float* kvl = s.d_kv + (size_t)layer * s.kv_layer_stride;
    if constexpr (HD == 32 || HD == 64 || HD == 128) {
        const size_t smem = (size_t)(64 * (HD + 4) * 2 + 64 * HD + 64 * 68) * 4;
        s.stats.kernel_launches++;
        launch_pdl(k_attn_prefill_rt<HD>, dim3(nblk, m.H), 256, smem, s.stream, s.d_q, kvl, s.kv_slot_stride, s.v_offset, m.H,
                                                                        m.ctx, scale, qblk, s.d_att);
        return;
    }
    size_t smem = (size_t)(64 * (HD + 1) * 2 + 64 * HD + 64 * 65) * 4;
    s.stats.kernel_launches++; launch_pdl(k_attn_prefill<HD>, dim3(nblk, m.H), 256, smem, s.stream, s.d_q, kvl, s.kv_slot_stride, s.v_offset, m.H,
                                                                 m.ctx, scale, qblk, s.d_att);
}

// Query blocks of the prefill attention: <= 64 rows for the SIMT kernels,
// <= 128 rows (may be null) for the tensor-core kernel.
struct QBlocks {
    int n;
    const int4* b;
    int n2;
    const int4* b2;
};

// ctx_hi / ctx_lo (optional): where the tensor-core kernel writes the TF32
// halves of the result instead of s.d_att; returns whether it did.
static bool launch_attn_prefill(DeviceSession& s, QBlocks qb, int layer, float* ctx_hi = nullptr,
                                float* ctx_lo = nullptr) {
    const fb2_model& m = *s.model;
    if (s.dm->attn_tc && s.dm->tc_ok && s.d_tc_err && qb.b2 && qb.n2 > 0) {
        const float* kvl = s.d_kv + (size_t)layer * s.kv_layer_stride;
        s.stats.kernel_launches++;
        launch_pdl(k_attn_prefill_tc, dim3(qb.n2, m.H), ATC_THREADS, (size_t)ATC_SMEM, s.stream, s.d_q, kvl,
                   s.kv_slot_stride, s.v_offset, m.H, m.ctx, 1.0f / sqrtf((float)m.hd), qb.b2,
                   ctx_lo ? ctx_hi : s.d_att, s.d_tc_err, ctx_lo);
        return ctx_lo != nullptr;
    }
    const int nblk = qb.n;
    const int4* qblk = qb.b;
    switch (s.model->hd) {
    case 4: launch_attn_prefill_hd<4>(s, nblk, qblk, layer); break;
    case 8: launch_attn_prefill_hd<8>(s, nblk, qblk, layer); break;
    case 16: launch_attn_prefill_hd<16>(s, nblk, qblk, layer); break;
    case 32: launch_attn_prefill_hd<32>(s, nblk, qblk, layer); break;
    case 64: launch_attn_prefill_hd<64>(s, nblk, qblk, layer); break;
    case 128: launch_attn_prefill_hd<128>(s, nblk, qblk, layer); break;
    default: fail(FB2_UNSUPPORTED, "head_dim must be a power of two in [4, 128]");
    }
    return false;
}

static void launch_head(DeviceSession& s, int M, const float* xln, const int* out_slot_host_unused,
                        float* logits_base) {
    (void)out_slot_host_unused;
    const fb2_model& m = *s.model;
    // batches of rows: one pass over tok_emb on the tensor cores (bf16
    // weights: the decode-batch GEMM reads the bf16 rows once)
    if (M > kMaxGemvRows && s.dm->tc_ok && s.d_ahi && !(s.dm->bf16 && M >= kTcMinRows)) {
        Epi e = make_epi(EPI_BIAS, s.dm->tc_head_blob + 2 * (size_t)m.V * m.D, nullptr, logits_base);
        if (launch_gemm_tc(s.stream, s.dm->sm_count, M, m.D, m.V, xln, s.d_ahi, s.d_alo, s.dm->tc_head_maps, e,
                           s.d_tc_err, s.d_tc_part, s.tc_part_cap, &s.stats.kernel_launches, s.dm->bf16))
            return;
    }
    int blocks = std::min(ceil_div(m.V, 8), 8 * s.dm->sm_count);
    for (int m0 = 0; m0 < M; m0 += kMaxGemvRows) {
        int mm = std::min(kMaxGemvRows, M - m0);
        const float* x = xln + (size_t)m0 * m.D;
        float* out = logits_base + (size_t)m0 * m.V;
        size_t smem;
#define HEAD_CASE(R)                                                                               \
    if (mm <= R) {                                                                                 \
        smem = (size_t)R * m.D * 4;                                                                \
        s.stats.kernel_launches++;                                                                 \
        if (s.dm->bf16)                                                                            \
            launch_pdl(k_head<R, WBF16>, blocks, 256, smem, s.stream, mm, m.D, m.V, x, s.dm->w16.at(s.dm->tok_emb), out, m.V); \
        else                                                                                       \
            launch_pdl(k_head<R>, blocks, 256, smem, s.stream, mm, m.D, m.V, x, s.dm->tok_emb, out, m.V);  \
        continue;                                                                                  \
    }
        HEAD_CASE(1) HEAD_CASE(2) HEAD_CASE(4) HEAD_CASE(8) HEAD_CASE(16)
#undef HEAD_CASE
    }
}

// All transformer blocks (TransformerBlock.Forward, Layers.cs:384-392) over
// rows 0..M-1 of d_x.  decode: single-row attention over the cache;
// otherwise causal prefill attention over the query blocks.
static void run_layers(DeviceSession& s, int M, Rows R, bool decode, QBlocks qb) {
    const fb2_model& m = *s.model;
    for (int l = 0; l < m.L; l++) {
        const LayerW& w = s.dm->layers[l];
        Epi eq = make_epi(EPI_QKV, w.qkv_b, nullptr, s.d_q);
        eq.kv_layer = s.d_kv + (size_t)l * s.kv_layer_stride;
        eq.kv_slot_stride = s.kv_slot_stride;
        eq.v_offset = s.v_offset;
        eq.D = m.D;
        eq.hd = m.hd;
        eq.ctx = m.ctx;
        eq.R = R;
        const CUtensorMap* tcm = s.dm->tc_ok ? s.dm->tc_maps[l].data() : nullptr;
        if (!decode && tcm && s.d_ahi2 && M >= kTcMinRows) {
            // prefill on the tensor cores: LN1, the attention, LN2 and fc write
            // their outputs as the next GEMM's TF32 halves (no split kernels)
            launch_layernorm(s, M, s.d_x, w.ln1_w, w.ln1_b, s.d_ahi, nullptr, s.d_alo);
            launch_linear_split(s, M, m.D, 3 * m.D, s.d_ahi, s.d_alo, tcm, eq);
            const Epi ep = make_epi(EPI_RESID, w.proj_b, s.d_x, s.d_x2);
            if (launch_attn_prefill(s, qb, l, s.d_ahi, s.d_alo)) launch_linear_split(s, M, m.D, m.D, s.d_ahi, s.d_alo, tcm + 3, ep);
            else launch_linear(s, M, m.D, m.D, s.d_att, w.proj_w, ep, tcm + 3);
            launch_layernorm(s, M, s.d_x2, w.ln2_w, w.ln2_b, s.d_ahi, nullptr, s.d_alo);
            Epi ef = make_epi(EPI_GELU_SPLIT, w.fc_b, nullptr, s.d_ahi2);
            ef.out_lo = s.d_alo2;
            launch_linear_split(s, M, m.D, m.F, s.d_ahi, s.d_alo, tcm + 6, ef);
            launch_linear_split(s, M, m.F, m.D, s.d_ahi2, s.d_alo2, tcm + 9, make_epi(EPI_RESID, w.mproj_b, s.d_x2, s.d_x));
            continue;
        }
        launch_layernorm(s, M, s.d_x, w.ln1_w, w.ln1_b, s.d_ln, nullptr);
        launch_linear(s, M, m.D, 3 * m.D, s.d_ln, w.qkv_w, eq, tcm);
        if (decode) launch_attn_decode(s, M, l, R);
        else launch_attn_prefill(s, qb, l);
        launch_linear(s, M, m.D, m.D, s.d_att, w.proj_w, make_epi(EPI_RESID, w.proj_b, s.d_x, s.d_x2), tcm ? tcm + 3 : nullptr);
        launch_layernorm(s, M, s.d_x2, w.ln2_w, w.ln2_b, s.d_ln, nullptr);
        launch_linear(s, M, m.D, m.F, s.d_ln, w.fc_w, make_epi(EPI_GELU, w.fc_b, nullptr, s.d_h), tcm ? tcm + 6 : nullptr);
        launch_linear(s, M, m.F, m.D, s.d_h, w.mproj_w, make_epi(EPI_RESID, w.mproj_b, s.d_x2, s.d_x), tcm ? tcm + 9 : nullptr);
    }
}

// One KV-cached decode step for slots 0..n-1 (graph-captured).
static void enqueue_decode_step(DeviceSession& s, int n) {
    const fb2_model& m = *s.model;
    s.stats.kernel_launches++; launch_pdl(k_step_prepare, ceil_div(n, 128), 128, 0, s.stream, n, s.d_len, s.d_done, m.ctx, s.d_row_seq, s.d_row_pos,
                                                          s.d_row_hidx, s.d_row_active);
    Rows R{s.d_row_seq, s.d_row_pos, s.d_row_hidx, s.d_row_active};
    s.stats.kernel_launches++; launch_pdl(k_embed, n, 128, 0, s.stream, n, R, s.d_hist, s.hist_cap, s.dm->tok_emb, s.dm->pos_emb, m.D, m.V, s.d_x);
    run_layers(s, n, R, true, QBlocks{0, nullptr, 0, nullptr});
    launch_layernorm(s, n, s.d_x, s.dm->lnf_w, s.dm->lnf_b, s.d_lnf, nullptr);
    launch_head(s, n, s.d_lnf, nullptr, s.d_logits);
}

static void run_decode_step(DeviceSession& s, int n) {
    if (s.graph && (s.graph_n != n)) {
        cudaGraphExecDestroy(s.graph);
        s.graph = nullptr;
    }
    if (!s.graph) {
        cudaGraph_t g = nullptr;
        const long long before = s.stats.kernel_launches;
        CK(cudaStreamBeginCapture(s.stream, cudaStreamCaptureModeThreadLocal));
        try {
            enqueue_decode_step(s, n);
            s.graph_kernels = s.stats.kernel_launches - before;
            s.stats.kernel_launches = before;
        } catch (...) {
            cudaStreamEndCapture(s.stream, &g);
            if (g) cudaGraphDestroy(g);
            throw;
        }
        CK(cudaStreamEndCapture(s.stream, &g));
        cudaError_t e = cudaGraphInstantiate(&s.graph, g, 0);
        cudaGraphDestroy(g);
        CK(e);
        s.graph_n = n;
    }
    CK(cudaGraphLaunch(s.graph, s.stream));
    s.stats.kernel_launches += s.graph_kernels;
    s.stats.decode_steps++;
}

// Whether k_decode_mega can run a decode of n rows with these options: up to
// 8 rows, greedy or top-k <= 64 (the candidate union stays small).
static bool mk_eligible(const DeviceSession& s, int n, const fb2_sampling& sp) {
    if (!s.mk_use || n < 1 || n > MK_MAX_ROWS) return false;
    if (sp.temperature > 0.0f && !(sp.top_k > 0 && sp.top_k <= MK_MAX_TOPK && sp.top_k < s.model->V)) return false;
    return true;
}

// One launch of k_decode_mega: `nsteps` decode steps for slots 0..n-1, none
// of which may slide within them.  Cooperative launch: one CTA per SM, all
// resident (the kernel's CTAs wait on one another).
static void run_mega(DeviceSession& s, int n, int nsteps, const SampleParams& P, const double* d_uni, int* d_out,
                     int out_stride, bool bookkeep) {
    const fb2_model& m = *s.model;
    const DeviceModel& dm = *s.dm;
    const int MR = n <= 1 ? 1 : n <= 2 ? 2 : n <= 4 ? 4 : 8;
    const int nW = dm.mk_nW;
    const int hc_cs = dm.mk_hc ? dm.mk_cs : 0;
    // head-cluster path: 32 KB stages (fewer per-stage waits) when at least
    // five fit next to the rest, else 16 KB
    int sb = MK_STAGE;
    int nstage = 0;
    if (dm.mk_hc) {
        nstage = mk_nstage(m, MR, nW, s.device, hc_cs, MK_STAGE_HC);
        if (nstage >= 5) sb = MK_STAGE_HC;
    }
    if (sb == MK_STAGE) nstage = mk_nstage(m, MR, nW, s.device, hc_cs, MK_STAGE);
    if (nstage == 0) fail(FB2_UNSUPPORTED, "persistent decode kernel does not fit shared memory");
    MkArgs a{};
    a.V = m.V; a.ctx = m.ctx; a.D = m.D; a.L = m.L; a.H = m.H; a.hd = m.hd; a.F = m.F;
    a.nW = nW; a.nstage = nstage; a.slice_max = mk_slice_max(m.V, nW);
    a.layers = dm.d_mk_layers;
    a.tok_emb = dm.tok_emb; a.pos_emb = dm.pos_emb; a.lnf_w = dm.lnf_w; a.lnf_b = dm.lnf_b;
    a.kv = s.d_kv; a.kv_slot_stride = s.kv_slot_stride; a.kv_layer_stride = s.kv_layer_stride; a.v_offset = s.v_offset;
    a.hist = s.d_hist; a.hist_stride = s.hist_cap;
    a.len = s.d_len; a.count = s.d_count; a.done = s.d_done;
    a.uniforms = d_uni; a.uni_stride = P.max_new > 0 ? P.max_new : 1;
    a.out_tokens = d_out; a.out_stride = out_stride;
    a.logits_out = s.d_logits;
    a.sp = P;
    a.n_rows = n;
    a.row_slot = s.mk_rows;
    a.bookkeep = bookkeep ? 1 : 0;
    a.xq = s.mk_xq; a.xkv = s.mk_xkv; a.xx2 = s.mk_xx2; a.xh = s.mk_xh; a.xx = s.mk_xx;
    a.xpart = s.mk_xpart; a.cand_hdr = s.mk_hdr; a.xacc = s.mk_xacc; a.maxc = mk_maxc(m.ctx, m.hd);
    a.cand_val = s.mk_cval; a.cand_idx = s.mk_cidx;
    a.stepdone = s.mk_stepdone; a.err = s.mk_err;
    a.gstep0 = s.mk_gstep; a.nsteps = nsteps;
    a.trace = s.mk_trace; a.trace_steps = s.mk_trace_steps;
    a.timeout_ns = MK_TIMEOUT_NS;
    a.withhold_cta = -1;
    if (s.test_withhold_cta >= 0) {  // one launch only
        a.timeout_ns = s.test_wait_ns;
        a.withhold_cta = s.test_withhold_cta;
        s.test_withhold_cta = -1;
    }
    {
        const char* ps = getenv("FORGE_B200_MK_PSLEEP");
        a.prod_sleep_ns = ps ? (unsigned)atoi(ps) : 200u;
    }
    a.stage_bytes = sb;
    a.hc = dm.mk_hc ? 1 : 0;
    a.cs = dm.mk_hc ? dm.mk_cs : 1;
    a.nhead = dm.mk_hc ? dm.mk_nhead : 0;
    a.acc = s.mk_acc;
    const size_t smem = mk_smem(m, MR, nW, nstage, hc_cs, sb);
    void* args[] = {&a};
    const void* f = mk_kernel(MR, dm.mk_hc);
    if (dm.mk_hc) {
        // clusters of mk_cs CTAs; cooperative, so the launch fails rather than
        // runs if not every CTA can be resident (the CTAs wait on one another)
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(nW);
        cfg.blockDim = dim3(MK_THREADS);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = s.stream;
        cudaLaunchAttribute at[2];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = dm.mk_cs;
        at[0].val.clusterDim.y = 1;
        at[0].val.clusterDim.z = 1;
        at[1].id = cudaLaunchAttributeCooperative;
        at[1].val.cooperative = 1;
        cfg.attrs = at;
        // FORGE_B200_MK_COOP=0 (profiling only: Nsight Compute does not launch
        // cooperative cluster grids) drops the residency check; the plan's
        // cluster count is within the device's active-cluster limit, and a
        // grid that is not fully resident ends in the waits' timeout status.
        const char* coop = getenv("FORGE_B200_MK_COOP");
        cfg.numAttrs = coop && coop[0] == '0' ? 1 : 2;
        CK(cudaLaunchKernelExC(&cfg, f, args));
    } else {
        CK(cudaLaunchCooperativeKernel(f, dim3(nW), dim3(MK_THREADS), args, smem, s.stream));
    }
    s.stats.kernel_launches++;
    s.stats.decode_steps += nsteps;
    s.stats.persistent_steps += nsteps;
    s.mk_gstep += nsteps;
}

// Host check of the persistent kernel's error flag (after a synchronize);
// resets its state and fails with FB2_TIMEOUT when a bounded wait expired.
static void mk_check(DeviceSession& s) {
    if (s.d_tc_err) {  // tensor-core GEMM: a bounded wait expired
        int terr = 0;
        CK(cudaMemcpy(&terr, s.d_tc_err, sizeof(int), cudaMemcpyDeviceToHost));
        if (terr != 0) {
            CK(cudaMemset(s.d_tc_err, 0, sizeof(int)));
            fail(FB2_TIMEOUT, "tensor-core GEMM: a bounded wait expired (code " + std::to_string(terr) + ")");
        }
    }
    if (!s.mk_use) return;
    int err = 0;
    CK(cudaMemcpy(&err, s.mk_err, sizeof(int), cudaMemcpyDeviceToHost));
    if (err != 0) {
        mk_reset(s);
        CK(cudaStreamSynchronize(s.stream));
        if (err == MK_ERR_LAYOUT) fail(FB2_CUDA_ERROR, "persistent decode kernel: shared-memory layout not 16-byte aligned");
        fail(FB2_TIMEOUT, "persistent decode kernel: a bounded wait expired (code " + std::to_string(err) + ")");
    }
}

// Prefill of one chunk: rows described by the uploaded tables.
// tab layout per chunk: row_seq[rows], row_pos[rows], qblk (int4) [nqblk],
// qblk2 (int4) [nqblk2],
// last_row[nslots], out_slot[nslots].
struct PrefillTables {
    const int* row_seq;
    const int* row_pos;
    const int4* qblk;
    const int* last_row;
    const int* out_slot;
};

__global__ void k_gather_logits_rows(int n, const int* out_slot, const float* src, float* dst, int V) {
    pdl_wait();
    // src rows are chunk-compact; dst rows are session slots
    int r = blockIdx.y;
    if (r >= n) return;
    const float* a = src + (size_t)r * V;
    float* b = dst + (size_t)out_slot[r] * V;
    for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < V; i += gridDim.x * blockDim.x) b[i] = a[i];
}

__global__ void k_prefill_hidx(int rows, const int* row_seq, const int* row_pos, const int* len, int ctx, int* hidx) {
    pdl_wait();
    int r = blockIdx.x * blockDim.x + threadIdx.x;
    if (r >= rows) return;
    int L = len[row_seq[r]];
    int w = L < ctx ? L : ctx;
    hidx[r] = L - w + row_pos[r];
}

static void run_prefill_chunk(DeviceSession& s, const ChunkPlan& c, const int* d_tab_base) {
    const fb2_model& m = *s.model;
    const int* row_seq = d_tab_base + c.row_off;
    const int* row_pos = row_seq + c.rows;
    const int4* qblk = reinterpret_cast<const int4*>(d_tab_base + c.qblk_off);
    const int4* qblk2 = reinterpret_cast<const int4*>(d_tab_base + c.qblk2_off);
    const int* last_row = d_tab_base + c.slot_off;
    const int* out_slot = last_row + c.nslots;
    s.stats.kernel_launches++; launch_pdl(k_prefill_hidx, ceil_div(c.rows, 256), 256, 0, s.stream, c.rows, row_seq, row_pos, s.d_len, m.ctx,
                                                               s.d_row_hidx);
    Rows R{row_seq, row_pos, s.d_row_hidx, s.d_ones};
    s.stats.kernel_launches++; launch_pdl(k_embed, c.rows, 128, 0, s.stream, c.rows, R, s.d_hist, s.hist_cap, s.dm->tok_emb, s.dm->pos_emb, m.D, m.V,
                                          s.d_x);
    run_layers(s, c.rows, R, false, QBlocks{c.nqblk, qblk, c.nqblk2, qblk2});
    launch_layernorm(s, c.nslots, s.d_x, s.dm->lnf_w, s.dm->lnf_b, s.d_lnf, last_row);
    // head into the chunk-compact area after the slots' logits, then scatter
    float* tmp = s.d_logits + (size_t)s.nslots * m.V;
    launch_head(s, c.nslots, s.d_lnf, nullptr, tmp);
    s.stats.kernel_launches++; launch_pdl(k_gather_logits_rows, dim3(std::min(ceil_div(m.V, 256), 64), c.nslots), 256, 0, s.stream, c.nslots, out_slot,
                                                                                              tmp, s.d_logits, m.V);
    s.stats.prefill_rows += c.rows;
}

// Builds prefill chunk tables for slots `order` with window lengths `wl`
// (slot-local indices), appending to `tab` and `plans`.  `start` (optional):
// per slot the first position to compute; the cache already holds K/V of
// the positions before it.
static void plan_prefill(const DeviceSession& s, const std::vector<int>& order, const std::vector<int>& wl,
                         std::vector<int>& tab, std::vector<ChunkPlan>& plans, const std::vector<int>* start = nullptr) {
    auto st = [&](int sl) { return start ? (*start)[sl] : 0; };
    size_t i = 0;
    while (i < order.size()) {
        size_t j = i;
        int rows = 0;
        while (j < order.size() && j - i < (size_t)kMaxChunkSlots &&
               (rows + wl[order[j]] - st(order[j]) <= s.row_cap || j == i)) {
            rows += wl[order[j]] - st(order[j]);
            j++;
        }
        if (rows > s.row_cap) fail(FB2_UNSUPPORTED, "window longer than the session's row capacity");
        ChunkPlan c{};
        c.rows = rows;
        c.nslots = (int)(j - i);
        c.row_off = (int)tab.size();
        std::vector<int> seq, pos;
        std::vector<int> q, q2;
        std::vector<int> last, slot;
        int r = 0;
        for (size_t k = i; k < j; k++) {
            const int sl = order[k], w = wl[sl], a = st(sl);
            for (int p = a; p < w; p++) {
                seq.push_back(sl);
                pos.push_back(p);
            }
            for (int p0 = a; p0 < w; p0 += 64) {
                int cnt = std::min(64, w - p0);
                q.push_back(r + (p0 - a));
                q.push_back(cnt);
                q.push_back(sl);
                q.push_back(p0);
            }
            for (int p0 = a; p0 < w; p0 += 128) {
                int cnt = std::min(128, w - p0);
                q2.push_back(r + (p0 - a));
                q2.push_back(cnt);
                q2.push_back(sl);
                q2.push_back(p0);
            }
            last.push_back(r + (w - a) - 1);
            slot.push_back(sl);
            r += w - a;
        }
        // tensor-core attention blocks, most keys first (the grid walks them in
        // order, so the short causal blocks fill the tail of the launch)
        {
            std::vector<std::array<int, 4>> b2(q2.size() / 4);
            for (size_t t = 0; t < b2.size(); t++) b2[t] = {q2[4 * t], q2[4 * t + 1], q2[4 * t + 2], q2[4 * t + 3]};
            std::stable_sort(b2.begin(), b2.end(), [](const std::array<int, 4>& x, const std::array<int, 4>& y) {
                return x[3] + x[1] > y[3] + y[1];
            });
            for (size_t t = 0; t < b2.size(); t++)
                for (int u = 0; u < 4; u++) q2[4 * t + u] = b2[t][u];
        }
        tab.insert(tab.end(), seq.begin(), seq.end());
        tab.insert(tab.end(), pos.begin(), pos.end());
        while (tab.size() % 4) tab.push_back(0);  // int4 alignment
        c.qblk_off = (int)tab.size();
        c.nqblk = (int)(q.size() / 4);
        tab.insert(tab.end(), q.begin(), q.end());
        c.qblk2_off = (int)tab.size();
        c.nqblk2 = (int)(q2.size() / 4);
        tab.insert(tab.end(), q2.begin(), q2.end());
        c.slot_off = (int)tab.size();
        tab.insert(tab.end(), last.begin(), last.end());
        tab.insert(tab.end(), slot.begin(), slot.end());
        while (tab.size() % 4) tab.push_back(0);
        plans.push_back(c);
        i = j;
    }
}

static void ensure_capacity(DeviceSession& s, int hist_cap_needed, size_t uni_needed, size_t out_needed) {
    DeviceGuard g(s.device);
    if (hist_cap_needed > s.hist_cap) {
        CK(cudaStreamSynchronize(s.stream));
        dfree(s.d_hist);
        s.hist_cap = std::max(hist_cap_needed, s.model->ctx + 64);
        s.d_hist = dalloc<int>((size_t)s.nslots * s.hist_cap);
        CK(cudaMemset(s.d_hist, 0, (size_t)s.nslots * s.hist_cap * sizeof(int)));
        if (s.graph) {  // the captured step embeds the history pointer and stride
            cudaGraphExecDestroy(s.graph);
            s.graph = nullptr;
        }
    }
    if (uni_needed > s.uni_cap) {
        CK(cudaStreamSynchronize(s.stream));
        dfree(s.d_uni);
        s.uni_cap = uni_needed;
        s.d_uni = dalloc<double>(s.uni_cap);
    }
    if (out_needed > s.out_cap) {
        CK(cudaStreamSynchronize(s.stream));
        dfree(s.d_out);
        s.out_cap = out_needed;
        s.d_out = dalloc<int>(s.out_cap);
    }
}

// Uploads `tab` (ints) + optional doubles through the pinned staging buffer.
static void upload_tables(DeviceSession& s, const std::vector<int>& tab, const std::vector<double>* uni) {
    size_t nint = tab.size();
    size_t nuni = uni ? uni->size() : 0;
    size_t bytes = nint * 4 + 16 + nuni * 8;
    if (s.tab_event_pending) {
        CK(cudaEventSynchronize(s.tab_event));
        s.tab_event_pending = false;
    }
    if (bytes > s.h_tab_cap) {
        if (s.h_tab) cudaFreeHost(s.h_tab);
        s.h_tab = nullptr;
        s.h_tab_cap = std::max(bytes, (size_t)1 << 16);
        CK(cudaMallocHost((void**)&s.h_tab, s.h_tab_cap));
    }
    if (nint > s.tab_cap) {
        CK(cudaStreamSynchronize(s.stream));
        dfree(s.d_tab);
        s.tab_cap = std::max(nint, (size_t)1024);
        s.d_tab = dalloc<int>(s.tab_cap);
    }
    if (nint) {
        memcpy(s.h_tab, tab.data(), nint * 4);
        CK(cudaMemcpyAsync(s.d_tab, s.h_tab, nint * 4, cudaMemcpyHostToDevice, s.stream));
    }
    if (nuni) {
        char* hu = reinterpret_cast<char*>(s.h_tab) + ((nint * 4 + 15) / 16) * 16;
        memcpy(hu, uni->data(), nuni * 8);
        CK(cudaMemcpyAsync(s.d_uni, hu, nuni * 8, cudaMemcpyHostToDevice, s.stream));
    }
    CK(cudaEventRecord(s.tab_event, s.stream));
    s.tab_event_pending = true;
}

__global__ void k_init_slots(int n, const int* __restrict__ plens_eff, const int* __restrict__ poff,
                             const int* __restrict__ ptok, int* hist, int hist_stride, int* len, int* count, int* done,
                             int max_new) {
    pdl_wait();
    int sidx = blockIdx.x;
    if (sidx >= n) return;
    int w = plens_eff[sidx];
    const int* src = ptok + poff[sidx];
    for (int i = threadIdx.x; i < w; i += blockDim.x) hist[(size_t)sidx * hist_stride + i] = src[i];
    if (threadIdx.x == 0) {
        len[sidx] = w;
        count[sidx] = 0;
        done[sidx] = max_new <= 0;
    }
}

// Device-pointer variant of the slot init: prompt tokens and lengths already
// on the device; keeps the last min(len, ctx) tokens of each prompt.
__global__ void k_init_slots_device(int n, const int* __restrict__ plens, const int* __restrict__ ptok, int ctx,
                                    int* hist, int hist_stride, int* len, int* count, int* done, int max_new) {
    pdl_wait();
    int sidx = blockIdx.x;
    if (sidx >= n) return;
    long long off = 0;
    for (int i = 0; i < sidx; i++) off += plens[i];
    int pl = plens[sidx];
    int w = pl < ctx ? pl : ctx;
    const int* src = ptok + off + (pl - w);
    for (int i = threadIdx.x; i < w; i += blockDim.x) hist[(size_t)sidx * hist_stride + i] = src[i];
    if (threadIdx.x == 0) {
        len[sidx] = w;
        count[sidx] = 0;
        done[sidx] = max_new <= 0;
    }
}

__global__ void k_copy_counts(int n, const int* count, int* out) {
    pdl_wait();
    int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i < n) out[i] = count[i];
}

static SampleParams to_params(const fb2_sampling& sp) {
    SampleParams p;
    p.temperature = sp.temperature;
    p.top_k = sp.top_k;
    p.penalty = sp.repetition_penalty;
    p.ngram = sp.no_repeat_ngram;
    p.eos = sp.eos_id;
    p.max_new = sp.max_new_tokens;
    return p;
}

static void validate_sampling(const fb2_model& m, const fb2_sampling* sp) {
    if (!sp) fail(FB2_INVALID_ARG, "sampling options are NULL");
    if (!std::isfinite(sp->temperature)) fail(FB2_INVALID_ARG, "Temperature must be finite.");
    if (sp->max_new_tokens < 0) fail(FB2_INVALID_ARG, "maxNewTokens must be >= 0.");
    if (sp->eos_id >= m.V) fail(FB2_INVALID_ARG, "EOS token must be inside the model vocabulary.");
    if (!std::isfinite(sp->repetition_penalty) || sp->repetition_penalty < 1.0f)
        fail(FB2_INVALID_ARG, "Repetition penalty must be finite and >= 1.");
    if (sp->no_repeat_ngram < 0) fail(FB2_INVALID_ARG, "No-repeat n-gram size must be >= 0.");
}

// ---------------------------------------------------------------------------
// The token loop for one device's share of the sequences.
// ---------------------------------------------------------------------------
struct ShardJob {
    int first;  // first global sequence index of this shard
    int n;      // sequences on this device
    const int* prompt_tokens;     // host, this shard's first prompt
    const int* prompt_lens;       // host
    const int* dev_prompt_tokens; // device variant
    const int* dev_prompt_lens;
    const fb2_sampling* sp;
    int rng_mode;
    const int32_t* seeds;
    const double* uniforms;       // host [n_total * max_new] or device
    bool device_io;
    int* out_tokens;              // host [n * max_new] or device
    int* out_counts;              // host [n] or device
    fb2_token_cb cb;
    void* user;
    fb2_uniform_cb ucb;           // FB2_RNG_CALLBACK
    void* ucb_user;
    std::mutex* cb_mutex;         // serialises both callbacks across device threads
    std::atomic<int>* stop;
};

static void run_generate_shard(DeviceSession& s, const ShardJob& job) {
    DeviceGuard guard(s.device);
    const fb2_model& m = *s.model;
    const fb2_sampling& sp = *job.sp;
    const int n = job.n, ctx = m.ctx, max_new = sp.max_new_tokens;
    if (n == 0) return;
    ensure_capacity(s, ctx + max_new + 1, (size_t)n * std::max(max_new, 1), (size_t)n * std::max(max_new, 1));
    const bool sampled = sp.temperature > 0.0f;

    // host-side plan: effective window lengths and when each slot starts sliding
    std::vector<int> wl0(n), plen(n);
    std::vector<long long> poff(n);
    long long off = 0;
    for (int i = 0; i < n; i++) {
        plen[i] = job.prompt_lens[i];
        wl0[i] = std::min(plen[i], ctx);
        poff[i] = off;
        off += plen[i];
    }
    // slot i re-prefills at every step >= slide_at[i] (window before
    // truncation = plen + step > ctx, Sampler.cs:93-94)
    std::vector<int> slide_at(n);
    for (int i = 0; i < n; i++) slide_at[i] = std::max(1, ctx - wl0[i] + 1);
    std::vector<int> order(n);
    for (int i = 0; i < n; i++) order[i] = i;
    std::stable_sort(order.begin(), order.end(), [&](int a, int b) { return slide_at[a] < slide_at[b]; });

    // cached prefixes: a slot whose cache holds the K/V of this prompt's first
    // tokens (the previous turn of a chat) computes only the new positions
    std::vector<int> start(n, 0);
    if (!job.device_io && (int)s.kv_tokens.size() >= n)
        for (int i = 0; i < n; i++) {
            const std::vector<int>& kv = s.kv_tokens[i];
            if (kv.empty() || plen[i] > ctx) continue;
            const int* p = job.prompt_tokens + poff[i];
            int c = 0;
            while (c < (int)kv.size() && c < plen[i] && kv[c] == p[c]) c++;
            start[i] = std::min(c, plen[i] - 1);  // at least one row yields the logits
            s.stats.reused_prefix_rows += start[i];
        }
    for (auto& kv : s.kv_tokens) kv.clear();  // rewritten below for the host path

    std::vector<int> tab;
    std::vector<ChunkPlan> init_plans, slide_plans_all;
    std::vector<int> all(n);
    for (int i = 0; i < n; i++) all[i] = i;
    plan_prefill(s, all, wl0, tab, init_plans, &start);
    // sliding re-prefill: every window is ctx rows; plan chunks over prefixes
    // of `order` (the set that slides only grows with the step).
    std::vector<int> wctx(n, ctx);
    // plan per prefix length lazily: prefixes change at most n times
    std::vector<int> prefix_sizes;
    for (int k = 1; k <= n; k++)
        if (k == n || slide_at[order[k]] != slide_at[order[k - 1]]) prefix_sizes.push_back(k);
    std::vector<std::vector<ChunkPlan>> slide_plans(prefix_sizes.size());
    int first_slide = slide_at[order[0]];
    if (max_new > first_slide) {
        for (size_t pi = 0; pi < prefix_sizes.size(); pi++) {
            int k = prefix_sizes[pi];
            if (slide_at[order[k - 1]] >= max_new) break;
            std::vector<int> sub(order.begin(), order.begin() + k);
            plan_prefill(s, sub, wctx, tab, slide_plans[pi]);
        }
    }
    // prompts: device variant copies on device; host variant appends to tab
    int ptok_off = 0, pl_off = 0, poff_off = 0;
    if (!job.device_io) {
        while (tab.size() % 4) tab.push_back(0);
        ptok_off = (int)tab.size();
        for (int i = 0; i < n; i++) {
            const int* p = job.prompt_tokens + poff[i] + (plen[i] - wl0[i]);
            tab.insert(tab.end(), p, p + wl0[i]);
        }
        pl_off = (int)tab.size();
        tab.insert(tab.end(), wl0.begin(), wl0.end());
        poff_off = (int)tab.size();
        int acc = 0;
        for (int i = 0; i < n; i++) {
            tab.push_back(acc);
            acc += wl0[i];
        }
    }
    // uniforms.  FB2_RNG_CALLBACK pulls them from the caller: all up front
    // when every sequence will emit max_new tokens (no EOS, no token
    // callback), else one step at a time, only for sequences still running
    // (`pull_per_step`; every step then synchronises with the host).
    const bool pull = sampled && job.rng_mode == FB2_RNG_CALLBACK;
    const bool pull_per_step = pull && (job.cb || sp.eos_id >= 0);
    auto draw = [&](int i) {
        std::lock_guard<std::mutex> lk(*job.cb_mutex);
        return job.ucb(job.ucb_user, job.first + i);
    };
    std::vector<double> uni;
    const double* d_uni = nullptr;
    if (sampled && max_new > 0) {
        if (job.rng_mode == FB2_RNG_UNIFORMS) {
            if (job.device_io) d_uni = job.uniforms;
            else uni.assign(job.uniforms, job.uniforms + (size_t)n * max_new);
        } else if (pull) {
            uni.assign((size_t)n * max_new, 0.0);
            if (!pull_per_step)
                for (int k = 0; k < max_new; k++)
                    for (int i = 0; i < n; i++) uni[(size_t)i * max_new + k] = draw(i);
        } else {
            uni.resize((size_t)n * max_new);
            for (int i = 0; i < n; i++) {
                DotNetRandom r = (job.rng_mode == FB2_RNG_SEEDS) ? DotNetRandom(job.seeds[job.first + i])
                                                                  : s.rngs[i];
                for (int k = 0; k < max_new; k++) uni[(size_t)i * max_new + k] = r.next_double();
            }
        }
        if (!d_uni) d_uni = s.d_uni;
    }
    upload_tables(s, tab, uni.empty() ? nullptr : &uni);
    CK(cudaEventRecord(s.ev0, s.stream));

    int* d_out = job.device_io ? job.out_tokens : s.d_out;
    if (job.device_io) {
        s.stats.kernel_launches++; launch_pdl(k_init_slots_device, n, 256, 0, s.stream, n, job.dev_prompt_lens, job.dev_prompt_tokens, ctx, s.d_hist,
                                                     s.hist_cap, s.d_len, s.d_count, s.d_done, max_new);
    } else {
        s.stats.kernel_launches++; launch_pdl(k_init_slots, n, 256, 0, s.stream, n, s.d_tab + pl_off, s.d_tab + poff_off, s.d_tab + ptok_off, s.d_hist,
                                              s.hist_cap, s.d_len, s.d_count, s.d_done, max_new);
    }
    CK(cudaGetLastError());
    SampleParams P = to_params(sp);
    size_t ssmem = sampler_smem_bytes(m.V);
    auto sample_all = [&]() {
        s.stats.kernel_launches++; launch_pdl(k_sample_step, n, kSampleThreads, ssmem, s.stream, n, s.d_logits, m.V, ctx, s.d_hist, s.hist_cap, s.d_len,
                                                              s.d_count, s.d_done, d_uni, max_new, P, d_out, max_new);
    };
    std::vector<int> h_tok, h_cnt, prev_cnt(n, 0);
    std::vector<char> running(n, 1);  // per-step mode: sequences that will sample the next step
    // per-step uniform pull: the draws for `step` of the running sequences,
    // copied into their table entries ahead of the step's sampling
    auto pull_step = [&](int step) {
        if (!pull_per_step) return;
        for (int i = 0; i < n; i++) {
            if (!running[i]) continue;
            double& u = uni[(size_t)i * max_new + step];
            u = draw(i);
            CK(cudaMemcpyAsync(s.d_uni + (size_t)i * max_new + step, &u, sizeof(double), cudaMemcpyHostToDevice,
                               s.stream));
        }
    };
    auto stream_callbacks = [&](int step) -> bool {
        // returns true when generation should stop
        CK(cudaStreamSynchronize(s.stream));
        h_cnt.resize(n);
        CK(cudaMemcpy(h_cnt.data(), s.d_count, n * sizeof(int), cudaMemcpyDeviceToHost));
        h_tok.resize((size_t)n * max_new);
        CK(cudaMemcpy(h_tok.data(), d_out, (size_t)n * max_new * sizeof(int), cudaMemcpyDeviceToHost));
        bool any_active = false;
        for (int i = 0; i < n; i++) {
            for (int k = prev_cnt[i]; k < h_cnt[i] && job.cb; k++) {
                int rc;
                {
                    std::lock_guard<std::mutex> lk(*job.cb_mutex);
                    rc = job.cb(job.user, job.first + i, step, h_tok[(size_t)i * max_new + k]);
                }
                if (rc != 0) job.stop->store(1);
            }
            prev_cnt[i] = h_cnt[i];
            bool eos_hit = sp.eos_id >= 0 && h_cnt[i] > 0 && h_tok[(size_t)i * max_new + h_cnt[i] - 1] == sp.eos_id;
            running[i] = !eos_hit && h_cnt[i] < max_new;
            if (running[i]) any_active = true;
        }
        return job.stop->load() != 0 || !any_active;
    };

    const bool per_step = job.cb || pull_per_step;  // the host sees every step's tokens
    if (max_new > 0) {
        pull_step(0);
        for (const ChunkPlan& c : init_plans) run_prefill_chunk(s, c, s.d_tab);
        sample_all();
        CK(cudaGetLastError());
        bool stop = per_step ? stream_callbacks(0) : false;
        int step = 1;
        // Persistent kernel for every step before the first slide: one launch
        // (a step per launch when a callback streams tokens; 64-step launches
        // with an EOS so finished batches stop early).
        if (!stop && mk_eligible(s, n, sp)) {
            const int mk_end = std::min(max_new, slide_at[order[0]]);
            while (step < mk_end && !stop) {
                int ns = mk_end - step;
                if (per_step) ns = 1;
                else if (sp.eos_id >= 0) ns = std::min(ns, 64);
                pull_step(step);
                run_mega(s, n, ns, P, d_uni, d_out, max_new, true);
                step += ns;
                if (per_step) stop = stream_callbacks(step - 1);
                else if (sp.eos_id >= 0 && step < mk_end) {
                    std::vector<int> hd(n);
                    CK(cudaMemcpyAsync(hd.data(), s.d_done, n * sizeof(int), cudaMemcpyDeviceToHost, s.stream));
                    CK(cudaStreamSynchronize(s.stream));
                    bool all_done = true;
                    for (int i = 0; i < n; i++) all_done = all_done && hd[i];
                    if (all_done) stop = true;
                }
            }
        }
        for (; step < max_new && !stop; step++) {
            // slots with slide_at <= step re-prefill; the rest decode
            int k = 0;
            while (k < n && slide_at[order[k]] <= step) k++;
            pull_step(step);
            if (k < n) run_decode_step(s, n);
            if (k > 0) {
                size_t pi = 0;
                while (prefix_sizes[pi] < k) pi++;
                for (const ChunkPlan& c : slide_plans[pi]) run_prefill_chunk(s, c, s.d_tab);
                s.stats.reprefills += k;
            }
            sample_all();
            if (per_step) stop = stream_callbacks(step);
            else if (sp.eos_id >= 0 && (step % 64) == 0) {
                // all slots finished? (cheap poll, keeps the pipeline mostly full)
                std::vector<int> hd(n);
                CK(cudaMemcpyAsync(hd.data(), s.d_done, n * sizeof(int), cudaMemcpyDeviceToHost, s.stream));
                CK(cudaStreamSynchronize(s.stream));
                bool all_done = true;
                for (int i = 0; i < n; i++) all_done = all_done && hd[i];
                if (all_done) break;
            }
        }
    }
    CK(cudaGetLastError());
    CK(cudaEventRecord(s.ev1, s.stream));
    if (job.device_io) {
        s.stats.kernel_launches++; launch_pdl(k_copy_counts, ceil_div(n, 128), 128, 0, s.stream, n, s.d_count, job.out_counts);
        CK(cudaGetLastError());
        return;
    }
    // results back to the host
    std::vector<int> counts(n);
    CK(cudaMemcpyAsync(counts.data(), s.d_count, n * sizeof(int), cudaMemcpyDeviceToHost, s.stream));
    if (max_new > 0)
        CK(cudaMemcpyAsync(job.out_tokens, d_out, (size_t)n * max_new * sizeof(int), cudaMemcpyDeviceToHost, s.stream));
    CK(cudaStreamSynchronize(s.stream));
    mk_check(s);
    float ms = 0.f;
    if (cudaEventElapsedTime(&ms, s.ev0, s.ev1) == cudaSuccess) s.stats.decode_ms += ms;
    for (int i = 0; i < n; i++) {
        job.out_counts[i] = counts[i];
        s.stats.tokens_generated += counts[i];
        if (job.rng_mode == FB2_RNG_SESSION && sampled)
            for (int k = 0; k < counts[i]; k++) s.rngs[i].next_double();
    }
    // the cache now holds the K/V of the prompt and of every generated token
    // but the last (never fed), at positions 0.. when the window never slid
    if ((int)s.kv_tokens.size() < n) s.kv_tokens.resize(n);
    for (int i = 0; i < n; i++) {
        const int fed = plen[i] + std::max(counts[i] - 1, 0);
        if (plen[i] == 0 || fed > ctx) continue;
        std::vector<int>& kv = s.kv_tokens[i];
        kv.assign(job.prompt_tokens + poff[i], job.prompt_tokens + poff[i] + plen[i]);
        if (max_new > 0)
            kv.insert(kv.end(), job.out_tokens + (size_t)i * max_new, job.out_tokens + (size_t)i * max_new + std::max(counts[i] - 1, 0));
    }
}

// ---------------------------------------------------------------------------
// Scratch for fb2_forward_last_logits_noalloc: one file-scope device array
// (8 MiB on every GPU that loads this library, held until the process
// exits).  Host code must not use `g_noalloc_scratch` as a pointer: its
// device address comes from cudaGetSymbolAddress, taken once per device.
// ---------------------------------------------------------------------------
constexpr size_t kNoallocScratchFloats = (size_t)2 << 20;  // 8 MiB
constexpr int kNoallocMaxRows = 16;                         // window length limit
static __device__ __align__(256) float g_noalloc_scratch[kNoallocScratchFloats];

namespace {
std::mutex g_noalloc_mutex;
float* g_noalloc_ptr[256] = {};  // device address of the scratch, per device ordinal

// Layout of the scratch for one window of n <= kNoallocMaxRows tokens.
struct NoallocLayout {
    size_t x, x2, ln, q, att, h, lnf, kv, part, tickets, ints, total;
};
NoallocLayout noalloc_layout(const fb2_model& m) {
    auto up = [](size_t v) { return (v + 63) / 64 * 64; };  // 256-byte aligned regions
    const size_t R = kNoallocMaxRows, D = m.D, F = m.F;
    NoallocLayout L{};
    size_t o = 0;
    L.x = o; o += up(R * D);
    L.x2 = o; o += up(R * D);
    L.ln = o; o += up(R * D);
    L.q = o; o += up(R * D);
    L.att = o; o += up(R * D);
    L.h = o; o += up(R * F);
    L.lnf = o; o += up((size_t)kMaxChunkSlots * D);
    L.kv = o; o += up((size_t)m.L * 2 * m.H * R * m.hd);
    L.part = o; o += up((size_t)512 * 1024);
    L.tickets = o; o += up(4096);
    L.ints = o; o += up(8 * R + 64);
    L.total = o;
    return L;
}
}  // namespace

// Window tables for one sequence of n tokens: rows 0..n-1 at positions
// 0..n-1, one query block, last row n-1 written to output row 0; tickets
// cleared (the array keeps the previous call's contents).
__global__ void k_noalloc_tables(int n, int* ints, unsigned int* tickets) {
    pdl_wait();
    int* row_seq = ints;
    int* row_pos = ints + kNoallocMaxRows;
    int* hidx = ints + 2 * kNoallocMaxRows;
    int* ones = ints + 3 * kNoallocMaxRows;
    int4* qblk = reinterpret_cast<int4*>(ints + 4 * kNoallocMaxRows);
    int* last_row = ints + 4 * kNoallocMaxRows + 4;
    int* out_slot = last_row + 1;
    int* len = last_row + 2;
    for (int i = threadIdx.x; i < 4096; i += blockDim.x) tickets[i] = 0u;
    for (int i = threadIdx.x; i < kNoallocMaxRows; i += blockDim.x) {
        row_seq[i] = 0;
        row_pos[i] = i;
        hidx[i] = i;
        ones[i] = 1;
    }
    if (threadIdx.x == 0) {
        *qblk = make_int4(0, n, 0, 0);
        *last_row = n - 1;
        *out_slot = 0;
        *len = n;
    }
}

// ---------------------------------------------------------------------------
// C ABI
// ---------------------------------------------------------------------------
extern "C" {

int32_t fb2_version(void) { return FB2_ABI_VERSION; }

const char* fb2_last_error(void) { return g_last_error.c_str(); }

int32_t fb2_device_count(int32_t* n) {
    return guarded([&] {
        if (!n) fail(FB2_INVALID_ARG, "n is NULL");
        int c = 0;
        cudaError_t e = cudaGetDeviceCount(&c);
        if (e != cudaSuccess) {
            cudaGetLastError();
            c = 0;
        }
        *n = c;
    });
}

int32_t fb2_model_create(const fb2_model_desc* desc, const float* const* params, int32_t n_params,
                         const int32_t* devices, int32_t n_devices, fb2_model** out) {
    return guarded([&] {
        if (!desc || !params || !out) fail(FB2_INVALID_ARG, "NULL argument");
        *out = nullptr;
        const fb2_model_desc& d = *desc;
        if (d.vocab_size <= 0 || d.context_length <= 0 || d.d_model <= 0 || d.n_layers <= 0 || d.n_heads <= 0)
            fail(FB2_INVALID_ARG, "model sizes must be positive");
        if (d.d_model % d.n_heads != 0) fail(FB2_INVALID_ARG, "DModel must be divisible by NHeads.");
        int hd = d.d_model / d.n_heads;
        if (hd < 4 || hd > 128 || (hd & (hd - 1))) fail(FB2_UNSUPPORTED, "head_dim must be a power of two in [4, 128]");
        if (d.d_model % 4 != 0 || d.d_model > 2048) fail(FB2_UNSUPPORTED, "d_model must be a multiple of 4, <= 2048");
        if (sampler_smem_bytes(d.vocab_size) > 227 * 1024)
            fail(FB2_UNSUPPORTED, "vocabulary too large for the on-chip sampler");
        if (d.weight_dtype != FB2_WEIGHTS_FP32 && d.weight_dtype != FB2_WEIGHTS_BF16)
            fail(FB2_INVALID_ARG, "weight_dtype must be FB2_WEIGHTS_FP32 or FB2_WEIGHTS_BF16");
        if (n_params != 4 + 12 * d.n_layers) fail(FB2_INVALID_ARG, "n_params must be 4 + 12*n_layers");
        for (int i = 0; i < n_params; i++)
            if (!params[i]) fail(FB2_INVALID_ARG, "parameter pointer is NULL");
        int ndev = 0;
        if (cudaGetDeviceCount(&ndev) != cudaSuccess || ndev == 0) {
            cudaGetLastError();
            fail(FB2_NO_DEVICE, "no CUDA device available");
        }
        std::vector<int> devs;
        if (!devices || n_devices <= 0) devs.push_back(0);
        else devs.assign(devices, devices + n_devices);
        auto m = new fb2_model();
        try {
            m->desc = d;
            m->V = d.vocab_size; m->ctx = d.context_length; m->D = d.d_model; m->L = d.n_layers;
            m->H = d.n_heads; m->hd = hd; m->F = 4 * d.d_model;
            std::vector<long long> numel = param_numels(d);
            // bf16 weights: tok_emb and the four projections of every layer,
            // rounded to nearest-even bf16 on the host before upload
            const bool bf16 = d.weight_dtype == FB2_WEIGHTS_BF16;
            std::vector<int> narrow_idx;
            if (bf16) {
                narrow_idx.push_back(0);
                for (int l = 0; l < d.n_layers; l++)
                    for (int j : {2, 4, 8, 10}) narrow_idx.push_back(2 + 12 * l + j);
            }
            std::vector<std::vector<float>> rounded(n_params);
            std::vector<const float*> up(params, params + n_params);
            for (int i : narrow_idx) {
                rounded[i].resize((size_t)numel[i]);
                for (long long k = 0; k < numel[i]; k++) rounded[i][k] = bf16_round_host(params[i][k]);
                up[i] = rounded[i].data();
            }
            std::vector<size_t> offs;
            size_t total = 0;
            for (long long k : numel) {
                offs.push_back(total);
                total += ((size_t)k + 63) / 64 * 64;  // 256-byte aligned tensors
            }
            for (int dev : devs) {
                if (dev < 0 || dev >= ndev) fail(FB2_INVALID_ARG, "device index out of range");
                DeviceGuard g(dev);
                cudaDeviceProp prop;
                CK(cudaGetDeviceProperties(&prop, dev));
                if (prop.major != 10) fail(FB2_UNSUPPORTED, "this build targets sm_100a (B200) only");
                configure_kernels(dev);
                DeviceModel dm;
                dm.device = dev;
                dm.sm_count = prop.multiProcessorCount;
                dm.blob = dalloc<float>(total);
                m->devs.push_back(dm);
                DeviceModel& D = m->devs.back();
                for (int i = 0; i < n_params; i++) {
                    CK(cudaMemcpy(D.blob + offs[i], up[i], (size_t)numel[i] * 4, cudaMemcpyHostToDevice));
                    D.p.push_back(D.blob + offs[i]);
                }
                if (bf16) {
                    D.bf16 = true;
                    size_t n16 = 0;
                    for (int i : narrow_idx) n16 += ((size_t)numel[i] + 127) / 128 * 128;
                    D.blob16 = dalloc<unsigned short>(n16);
                    size_t at = 0;
                    for (int i : narrow_idx) {
                        k_to_bf16_bits<<<(int)std::min<long long>(4096, (numel[i] + 255) / 256), 256>>>(D.p[i], numel[i],
                                                                                                  D.blob16 + at);
                        D.w16[D.p[i]] = D.blob16 + at;
                        at += ((size_t)numel[i] + 127) / 128 * 128;
                    }
                    CK(cudaGetLastError());
                    CK(cudaDeviceSynchronize());
                }
                D.tok_emb = D.p[0];
                D.pos_emb = D.p[1];
                for (int l = 0; l < d.n_layers; l++) {
                    const float* const* q = D.p.data() + 2 + 12 * l;
                    D.layers.push_back(LayerW{q[0], q[1], q[2], q[3], q[4], q[5], q[6], q[7], q[8], q[9], q[10], q[11]});
                }
                D.lnf_w = D.p[2 + 12 * d.n_layers];
                D.lnf_b = D.p[3 + 12 * d.n_layers];
                mk_setup(*m, D, up.data());
                tc_setup(*m, D);
            }
        } catch (...) {
            for (auto& dm : m->devs) {
                cudaSetDevice(dm.device);
                dfree(dm.blob);
                dfree(dm.relaid);
                dfree(dm.mk_fold);
                dfree(dm.d_mk_layers);
                dfree(dm.tc_blob);
                dfree(dm.tc_head_blob);
                dfree(dm.blob16);
            }
            delete m;
            throw;
        }
        *out = m;
    });
}

void fb2_model_destroy(fb2_model* m) {
    if (!m) return;
    for (auto& dm : m->devs) {
        cudaSetDevice(dm.device);
        dfree(dm.blob);
        dfree(dm.relaid);
        dfree(dm.mk_fold);
        dfree(dm.d_mk_layers);
        dfree(dm.tc_blob);
        dfree(dm.tc_head_blob);
        dfree(dm.blob16);
    }
    delete m;
}

int32_t fb2_session_create(fb2_model* m, int32_t max_seqs, fb2_session** out) {
    return guarded([&] {
        if (!m || !out) fail(FB2_INVALID_ARG, "NULL argument");
        if (max_seqs <= 0) fail(FB2_INVALID_ARG, "max_seqs must be positive");
        *out = nullptr;
        auto S = new fb2_session();
        S->model = m;
        S->max_seqs = max_seqs;
        try {
            int nd = (int)m->devs.size();
            int per = ceil_div(max_seqs, nd);
            for (int di = 0; di < nd; di++) {
                int slot0 = di * per, cnt = std::max(0, std::min(per, max_seqs - slot0));
                auto s = new DeviceSession();
                S->ds.push_back(s);
                s->model = m;
                s->dm = &m->devs[di];
                s->device = m->devs[di].device;
                s->slot0 = slot0;
                s->nslots = cnt;
                if (cnt == 0) continue;
                DeviceGuard g(s->device);
                CK(cudaStreamCreateWithFlags(&s->own_stream, cudaStreamNonBlocking));
                s->stream = s->own_stream;
                CK(cudaEventCreate(&s->ev0));
                CK(cudaEventCreate(&s->ev1));
                CK(cudaEventCreateWithFlags(&s->tab_event, cudaEventDisableTiming));
                const long long D = m->D, F = m->F;
                s->kv_layer_stride = 2LL * m->H * m->ctx * m->hd;
                s->v_offset = (long long)m->H * m->ctx * m->hd;
                s->kv_slot_stride = s->kv_layer_stride * m->L;
                s->d_kv = dalloc<float>((size_t)s->kv_slot_stride * cnt);
                s->d_len = dalloc<int>(cnt);
                s->d_count = dalloc<int>(cnt);
                s->d_done = dalloc<int>(cnt);
                CK(cudaMemset(s->d_len, 0, cnt * 4));
                CK(cudaMemset(s->d_count, 0, cnt * 4));
                CK(cudaMemset(s->d_done, 0, cnt * 4));
                s->hist_cap = m->ctx + 64;
                s->d_hist = dalloc<int>((size_t)cnt * s->hist_cap);
                CK(cudaMemset(s->d_hist, 0, (size_t)cnt * s->hist_cap * 4));
                // rows: enough for the largest prefill chunk
                long long want = (long long)cnt * m->ctx;
                s->row_cap = (int)std::max<long long>(m->ctx, std::min<long long>(want, 32768));
                s->row_cap = std::max(s->row_cap, cnt);
                size_t rc = s->row_cap;
                s->d_row_seq = dalloc<int>(rc);
                s->d_row_pos = dalloc<int>(rc);
                s->d_row_hidx = dalloc<int>(rc);
                s->d_row_active = dalloc<int>(rc);
                s->d_ones = dalloc<int>(rc);
                {
                    std::vector<int> ones(rc, 1);
                    CK(cudaMemcpy(s->d_ones, ones.data(), rc * 4, cudaMemcpyHostToDevice));
                }
                s->d_x = dalloc<float>(rc * D);
                s->d_x2 = dalloc<float>(rc * D);
                s->d_ln = dalloc<float>(rc * D);
                s->d_q = dalloc<float>(rc * D);
                s->d_att = dalloc<float>(rc * D);
                s->d_h = dalloc<float>(rc * F);
                if (s->dm->tc_ok) {
                    s->d_ahi = dalloc<float>(rc * F);
                    s->d_alo = dalloc<float>(rc * F);
                    s->d_ahi2 = dalloc<float>(rc * F);
                    s->d_alo2 = dalloc<float>(rc * F);
                    s->d_tc_err = dalloc<int>(1);
                    CK(cudaMemset(s->d_tc_err, 0, sizeof(int)));
                    s->tc_part_cap = (size_t)kTcSplitMax * 128 * (size_t)(4 * D);
                    s->d_tc_part = dalloc<float>(s->tc_part_cap);
                }
                s->d_logits = dalloc<float>((size_t)(cnt + kMaxChunkSlots) * m->V);
                s->d_lnf = dalloc<float>((size_t)std::max(cnt, kMaxChunkSlots) * D);
                s->attn_nsplit = ceil_div(m->ctx, kAttnChunk);
                s->d_attn_part = dalloc<float>((size_t)cnt * m->H * s->attn_nsplit * (m->hd + 2));
                s->gemv_part_cap = (size_t)64 * kMaxGemvRows * (size_t)std::max<long long>(4 * D, 1);
                s->d_gemv_part = dalloc<float>(s->gemv_part_cap);
                s->d_tickets = dalloc<unsigned int>(4096);
                CK(cudaMemset(s->d_tickets, 0, 4096 * 4));
                s->rngs.assign(cnt, DotNetRandom(0));
                s->stats.device_count = nd;
                mk_session_alloc(*s);
            }
        } catch (...) {
            for (auto s : S->ds) session_free(s);
            delete S;
            throw;
        }
        *out = S;
    });
}

void fb2_session_destroy(fb2_session* S) {
    if (!S) return;
    for (auto s : S->ds) session_free(s);
    delete S;
}

int32_t fb2_session_seed(fb2_session* S, int32_t seq, int32_t seed) {
    return guarded([&] {
        if (!S) fail(FB2_INVALID_ARG, "session is NULL");
        if (seq < 0 || seq >= S->max_seqs) fail(FB2_INVALID_ARG, "slot out of range");
        for (auto s : S->ds)
            if (seq >= s->slot0 && seq < s->slot0 + s->nslots) s->rngs[seq - s->slot0].reseed(seed);
    });
}

int32_t fb2_session_set_uniform_source(fb2_session* S, fb2_uniform_cb cb, void* user) {
    return guarded([&] {
        if (!S) fail(FB2_INVALID_ARG, "session is NULL");
        S->ucb = cb;
        S->ucb_user = cb ? user : nullptr;
    });
}

int32_t fb2_session_set_stream(fb2_session* S, int32_t device_slot, void* stream) {
    return guarded([&] {
        if (!S) fail(FB2_INVALID_ARG, "session is NULL");
        if (device_slot < 0 || device_slot >= (int)S->ds.size()) fail(FB2_INVALID_ARG, "device slot out of range");
        DeviceSession* s = S->ds[device_slot];
        s->stream = stream ? static_cast<cudaStream_t>(stream) : s->own_stream;
    });
}

static void check_generate_args(fb2_session* S, int32_t n_seqs, const int32_t* prompt_lens, const fb2_sampling* sp,
                                int32_t rng_mode, const int32_t* seeds, const void* uniforms) {
    if (!S) fail(FB2_INVALID_ARG, "session is NULL");
    if (n_seqs <= 0 || n_seqs > S->max_seqs) fail(FB2_INVALID_ARG, "n_seqs out of range");
    validate_sampling(*S->model, sp);
    if (prompt_lens)
        for (int i = 0; i < n_seqs; i++)
            if (prompt_lens[i] <= 0) fail(FB2_INVALID_ARG, "Need at least one prompt token.");
    if (rng_mode < FB2_RNG_SEEDS || rng_mode > FB2_RNG_CALLBACK) fail(FB2_INVALID_ARG, "bad rng_mode");
    if (sp->temperature > 0.0f && sp->max_new_tokens > 0) {
        if (rng_mode == FB2_RNG_SEEDS && !seeds) fail(FB2_INVALID_ARG, "seeds is NULL");
        if (rng_mode == FB2_RNG_UNIFORMS && !uniforms) fail(FB2_INVALID_ARG, "uniforms is NULL");
        if (rng_mode == FB2_RNG_CALLBACK && !S->ucb)
            fail(FB2_INVALID_ARG, "rng must not be null (FB2_RNG_CALLBACK without a uniform source)");
    }
}

static void run_shards(fb2_session* S, std::vector<ShardJob>& jobs) {
    std::vector<int> idx;
    for (size_t i = 0; i < jobs.size(); i++)
        if (jobs[i].n > 0) idx.push_back((int)i);
    if (idx.size() <= 1) {
        for (int i : idx) run_generate_shard(*S->ds[i], jobs[i]);
        return;
    }
    std::vector<std::thread> th;
    std::vector<int> st(jobs.size(), FB2_OK);
    std::vector<std::string> msg(jobs.size());
    for (int i : idx)
        th.emplace_back([&, i] {
            st[i] = guarded([&] { run_generate_shard(*S->ds[i], jobs[i]); });
            if (st[i] != FB2_OK) msg[i] = g_last_error;
        });
    for (auto& t : th) t.join();
    for (int i : idx)
        if (st[i] != FB2_OK) fail(st[i], msg[i]);
}

int32_t fb2_generate(fb2_session* S, int32_t n_seqs, const int32_t* prompt_tokens, const int32_t* prompt_lens,
                     const fb2_sampling* sp, int32_t rng_mode, const int32_t* seeds, const double* uniforms,
                     int32_t* out_tokens, int32_t* out_counts, fb2_token_cb cb, void* user) {
    return guarded([&] {
        if (!prompt_tokens || !prompt_lens || !out_counts) fail(FB2_INVALID_ARG, "NULL argument");
        check_generate_args(S, n_seqs, prompt_lens, sp, rng_mode, seeds, uniforms);
        if (sp->max_new_tokens > 0 && !out_tokens) fail(FB2_INVALID_ARG, "out_tokens is NULL");
        const fb2_model& m = *S->model;
        long long total = 0;
        for (int i = 0; i < n_seqs; i++) total += prompt_lens[i];
        for (long long i = 0; i < total; i++)
            if (prompt_tokens[i] < 0 || prompt_tokens[i] >= m.V)
                fail(FB2_INVALID_ARG, "Token id out of range [0," + std::to_string(m.V) + ").");
        const int max_new = sp->max_new_tokens;
        std::mutex cbm;
        std::atomic<int> stop{0};
        std::vector<ShardJob> jobs;
        long long toff = 0;
        for (auto s : S->ds) {
            ShardJob j{};
            j.first = s->slot0;
            j.n = std::max(0, std::min(s->nslots, n_seqs - s->slot0));
            j.prompt_tokens = prompt_tokens + toff;
            j.prompt_lens = prompt_lens + std::min(s->slot0, n_seqs);
            for (int i = 0; i < j.n; i++) toff += prompt_lens[s->slot0 + i];
            j.sp = sp;
            j.rng_mode = rng_mode;
            j.seeds = seeds;
            j.uniforms = uniforms ? uniforms + (size_t)std::min(s->slot0, n_seqs) * max_new : nullptr;
            j.device_io = false;
            j.out_tokens = out_tokens ? out_tokens + (size_t)std::min(s->slot0, n_seqs) * max_new : nullptr;
            j.out_counts = out_counts + std::min(s->slot0, n_seqs);
            j.cb = cb;
            j.user = user;
            j.ucb = S->ucb;
            j.ucb_user = S->ucb_user;
            j.cb_mutex = &cbm;
            j.stop = &stop;
            jobs.push_back(j);
        }
        if (max_new == 0) {
            for (int i = 0; i < n_seqs; i++) out_counts[i] = 0;
            return;
        }
        run_shards(S, jobs);
    });
}

// The slots' caches are about to be overwritten outside the generate path.
static void forget_cached_prefixes(fb2_session* S) {
    for (auto d : S->ds)
        for (auto& kv : d->kv_tokens) kv.clear();
}

int32_t fb2_generate_device(fb2_session* S, int32_t n_seqs, const int32_t* device_prompt_tokens,
                            const int32_t* device_prompt_lens, const int32_t* host_prompt_lens, const fb2_sampling* sp,
                            int32_t rng_mode, const int32_t* seeds, const double* device_uniforms,
                            int32_t* device_out_tokens, int32_t* device_out_counts) {
    return guarded([&] {
        if (!device_prompt_tokens || !device_prompt_lens || !host_prompt_lens || !device_out_counts)
            fail(FB2_INVALID_ARG, "NULL argument");
        check_generate_args(S, n_seqs, host_prompt_lens, sp, rng_mode, seeds, device_uniforms);
        if (rng_mode == FB2_RNG_CALLBACK) fail(FB2_INVALID_ARG, "FB2_RNG_CALLBACK needs fb2_generate");
        if (S->ds.size() != 1) fail(FB2_UNSUPPORTED, "fb2_generate_device needs a single-device session");
        if (sp->max_new_tokens > 0 && !device_out_tokens) fail(FB2_INVALID_ARG, "out_tokens is NULL");
        std::mutex cbm;
        std::atomic<int> stop{0};
        ShardJob j{};
        j.first = 0;
        j.n = n_seqs;
        j.prompt_lens = host_prompt_lens;
        j.dev_prompt_tokens = device_prompt_tokens;
        j.dev_prompt_lens = device_prompt_lens;
        j.sp = sp;
        j.rng_mode = rng_mode;
        j.seeds = seeds;
        j.uniforms = device_uniforms;
        j.device_io = true;
        j.out_tokens = device_out_tokens;
        j.out_counts = device_out_counts;
        j.cb = nullptr;
        j.cb_mutex = &cbm;
        j.stop = &stop;
        if (sp->max_new_tokens == 0) {
            DeviceGuard g(S->ds[0]->device);
            CK(cudaMemsetAsync(device_out_counts, 0, n_seqs * 4, S->ds[0]->stream));
            return;
        }
        run_generate_shard(*S->ds[0], j);
    });
}

__global__ void k_bump_len(int n, int* len) {
    pdl_wait();
    int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i < n) len[i] += 1;
}

// Loads whole token sequences into the slots' histories with len = `len0`.
static void load_histories(DeviceSession& s, int n, const int* tokens_host, int seq_len, int len0) {
    std::vector<int> tab;
    tab.assign(tokens_host, tokens_host + (size_t)n * seq_len);
    int pl_off = (int)tab.size();
    for (int i = 0; i < n; i++) tab.push_back(seq_len);
    int poff_off = (int)tab.size();
    for (int i = 0; i < n; i++) tab.push_back(i * seq_len);
    upload_tables(s, tab, nullptr);
    s.stats.kernel_launches++; launch_pdl(k_init_slots, n, 256, 0, s.stream, n, s.d_tab + pl_off, s.d_tab + poff_off, s.d_tab, s.d_hist, s.hist_cap,
                                          s.d_len, s.d_count, s.d_done, 1);
    std::vector<int> lens(n, len0);
    CK(cudaMemcpyAsync(s.d_len, lens.data(), n * 4, cudaMemcpyHostToDevice, s.stream));
    CK(cudaStreamSynchronize(s.stream));
}

int32_t fb2_forward_last_logits(fb2_session* S, int32_t n_seqs, const int32_t* tokens, const int32_t* lens,
                                float* out_logits) {
    return guarded([&] {
        if (!S || !tokens || !lens || !out_logits) fail(FB2_INVALID_ARG, "NULL argument");
        if (n_seqs <= 0 || n_seqs > S->max_seqs) fail(FB2_INVALID_ARG, "n_seqs out of range");
        forget_cached_prefixes(S);
        const fb2_model& m = *S->model;
        long long total = 0;
        for (int i = 0; i < n_seqs; i++) {
            if (lens[i] <= 0) fail(FB2_INVALID_ARG, "Need at least one token.");
            if (lens[i] > m.ctx) fail(FB2_INVALID_ARG, "Sequence length exceeds ContextLength.");
            total += lens[i];
        }
        for (long long i = 0; i < total; i++)
            if (tokens[i] < 0 || tokens[i] >= m.V) fail(FB2_INVALID_ARG, "Token id out of range.");
        long long toff = 0;
        for (auto sp : S->ds) {
            DeviceSession& s = *sp;
            int n = std::max(0, std::min(s.nslots, n_seqs - s.slot0));
            if (n == 0) continue;
            DeviceGuard g(s.device);
            ensure_capacity(s, m.ctx + 1, 1, 1);
            std::vector<int> wl(n), all(n), tab;
            for (int i = 0; i < n; i++) { wl[i] = lens[s.slot0 + i]; all[i] = i; }
            std::vector<ChunkPlan> plans;
            plan_prefill(s, all, wl, tab, plans);
            while (tab.size() % 4) tab.push_back(0);
            int ptok_off = (int)tab.size();
            long long cnt = 0;
            for (int i = 0; i < n; i++) cnt += wl[i];
            tab.insert(tab.end(), tokens + toff, tokens + toff + cnt);
            int pl_off = (int)tab.size();
            tab.insert(tab.end(), wl.begin(), wl.end());
            int poff_off = (int)tab.size();
            int acc = 0;
            for (int i = 0; i < n; i++) { tab.push_back(acc); acc += wl[i]; }
            toff += cnt;
            upload_tables(s, tab, nullptr);
            s.stats.kernel_launches++; launch_pdl(k_init_slots, n, 256, 0, s.stream, n, s.d_tab + pl_off, s.d_tab + poff_off, s.d_tab + ptok_off,
                                                  s.d_hist, s.hist_cap, s.d_len, s.d_count, s.d_done, 1);
            for (const ChunkPlan& c : plans) run_prefill_chunk(s, c, s.d_tab);
            CK(cudaGetLastError());
            CK(cudaMemcpyAsync(out_logits + (size_t)s.slot0 * m.V, s.d_logits, (size_t)n * m.V * 4,
                               cudaMemcpyDeviceToHost, s.stream));
            CK(cudaStreamSynchronize(s.stream));
        }
    });
}

int32_t fb2_teacher_forced_logits(fb2_session* S, int32_t n_seqs, const int32_t* tokens, int32_t len,
                                  int32_t prompt_len, float* out_logits) {
    return guarded([&] {
        if (!S || !tokens || !out_logits) fail(FB2_INVALID_ARG, "NULL argument");
        const fb2_model& m = *S->model;
        if (n_seqs <= 0 || n_seqs > S->max_seqs) fail(FB2_INVALID_ARG, "n_seqs out of range");
        if (prompt_len < 1 || len < prompt_len || len > m.ctx) fail(FB2_INVALID_ARG, "need 1 <= prompt_len <= len <= ctx");
        forget_cached_prefixes(S);
        for (long long i = 0; i < (long long)n_seqs * len; i++)
            if (tokens[i] < 0 || tokens[i] >= m.V) fail(FB2_INVALID_ARG, "Token id out of range.");
        const int steps = len - prompt_len + 1;
        for (auto sp : S->ds) {
            DeviceSession& s = *sp;
            int n = std::max(0, std::min(s.nslots, n_seqs - s.slot0));
            if (n == 0) continue;
            DeviceGuard g(s.device);
            ensure_capacity(s, m.ctx + 1, 1, 1);
            load_histories(s, n, tokens + (size_t)s.slot0 * len, len, prompt_len);
            std::vector<int> wl(n, prompt_len), all(n), tab;
            for (int i = 0; i < n; i++) all[i] = i;
            std::vector<ChunkPlan> plans;
            plan_prefill(s, all, wl, tab, plans);
            upload_tables(s, tab, nullptr);
            for (const ChunkPlan& c : plans) run_prefill_chunk(s, c, s.d_tab);
            fb2_sampling greedy{};
            greedy.temperature = 0.0f;
            greedy.repetition_penalty = 1.0f;
            greedy.eos_id = -1;
            greedy.max_new_tokens = 1;
            const bool mk = mk_eligible(s, n, greedy);
            for (int st = 0; st < steps; st++) {
                if (st > 0) {
                    s.stats.kernel_launches++; launch_pdl(k_bump_len, ceil_div(n, 128), 128, 0, s.stream, n, s.d_len);
                    if (mk) run_mega(s, n, 1, to_params(greedy), nullptr, nullptr, 1, false);
                    else run_decode_step(s, n);
                }
                CK(cudaGetLastError());
                for (int i = 0; i < n; i++)
                    CK(cudaMemcpyAsync(out_logits + (((size_t)(s.slot0 + i)) * steps + st) * m.V,
                                       s.d_logits + (size_t)i * m.V, (size_t)m.V * 4, cudaMemcpyDeviceToHost,
                                       s.stream));
            }
            CK(cudaStreamSynchronize(s.stream));
        }
    });
}

int32_t fb2_sample_logits(fb2_session* S, int32_t n, const float* logits, const int32_t* windows,
                          const int32_t* window_lens, const fb2_sampling* sp, const double* uniforms,
                          int32_t* out_ids) {
    return guarded([&] {
        if (!S || !logits || !window_lens || !out_ids) fail(FB2_INVALID_ARG, "NULL argument");
        if (n <= 0) fail(FB2_INVALID_ARG, "n must be positive");
        const fb2_model& m = *S->model;
        validate_sampling(m, sp);
        if (sp->temperature > 0.0f && !uniforms) fail(FB2_INVALID_ARG, "uniforms is NULL");
        long long wtot = 0;
        for (int i = 0; i < n; i++) {
            if (window_lens[i] < 0) fail(FB2_INVALID_ARG, "window length must be >= 0");
            wtot += window_lens[i];
        }
        if (wtot > 0 && !windows) fail(FB2_INVALID_ARG, "windows is NULL");
        DeviceSession& s = *S->ds[0];
        DeviceGuard g(s.device);
        std::vector<int> tab;
        tab.assign(windows ? windows : nullptr, windows ? windows + wtot : nullptr);
        int off_off = (int)tab.size();
        long long acc = 0;
        for (int i = 0; i < n; i++) { tab.push_back((int)acc); acc += window_lens[i]; }
        int len_off = (int)tab.size();
        tab.insert(tab.end(), window_lens, window_lens + n);
        int ids_off = (int)tab.size();
        for (int i = 0; i < n; i++) tab.push_back(0);
        std::vector<double> uni(n, 0.0);
        if (uniforms) uni.assign(uniforms, uniforms + n);
        ensure_capacity(s, 1, (size_t)n, 1);
        upload_tables(s, tab, &uni);
        float* d_l = dalloc<float>((size_t)n * m.V);
        try {
            CK(cudaMemcpyAsync(d_l, logits, (size_t)n * m.V * 4, cudaMemcpyHostToDevice, s.stream));
            s.stats.kernel_launches++; launch_pdl(k_sample_rows, n, kSampleThreads, sampler_smem_bytes(m.V), s.stream, 
                n, d_l, m.V, s.d_tab, s.d_tab + off_off, s.d_tab + len_off, s.d_uni, to_params(*sp), s.d_tab + ids_off);
            CK(cudaGetLastError());
            CK(cudaMemcpyAsync(out_ids, s.d_tab + ids_off, n * 4, cudaMemcpyDeviceToHost, s.stream));
            CK(cudaStreamSynchronize(s.stream));
        } catch (...) {
            cudaFree(d_l);
            throw;
        }
        cudaFree(d_l);
    });
}

int32_t fb2_init_params(const fb2_model_desc* desc, int32_t seed, float* const* params, int32_t n_params) {
    return guarded([&] {
        if (!desc || !params) fail(FB2_INVALID_ARG, "NULL argument");
        const fb2_model_desc& d = *desc;
        if (d.vocab_size <= 0 || d.context_length <= 0 || d.d_model <= 0 || d.n_layers <= 0 || d.n_heads <= 0)
            fail(FB2_INVALID_ARG, "model sizes must be positive");
        if (n_params != 4 + 12 * d.n_layers) fail(FB2_INVALID_ARG, "n_params must be 4 + 12*n_layers");
        std::vector<long long> numel = param_numels(d);
        DotNetRandom rng(seed);
        const float std_ = 0.02f;
        const float resid = 0.02f / sqrtf(2.0f * (float)d.n_layers);  // GptModel.cs:50
        auto normal = [&](float* p, long long n, float s) {  // Tensor.FillNormal, Tensor.cs:79-91
            for (long long i = 0; i < n; i += 2) {
                double u1 = 1.0 - rng.next_double();
                double u2 = rng.next_double();
                double r = std::sqrt(-2.0 * std::log(u1));
                p[i] = (float)(r * std::cos(2 * M_PI * u2) * (double)s);
                if (i + 1 < n) p[i + 1] = (float)(r * std::sin(2 * M_PI * u2) * (double)s);
            }
        };
        for (int i = 0; i < n_params; i++) {
            float* p = params[i];
            if (!p) fail(FB2_INVALID_ARG, "parameter pointer is NULL");
            long long n = numel[i];
            int kind = (i < 2) ? -1 : (i >= n_params - 2 ? 100 + (i - (n_params - 2)) : (i - 2) % 12);
            switch (kind) {
            case -1: case 2: case 8: normal(p, n, std_); break;
            case 4: case 10: normal(p, n, resid); break;
            case 0: case 6: case 100: std::fill(p, p + n, 1.0f); break;  // LayerNorm weights
            default: std::fill(p, p + n, 0.0f); break;                   // biases
            }
        }
    });
}

int32_t fb2_stats(fb2_session* S, fb2_stats_t* out) {
    return guarded([&] {
        if (!S || !out) fail(FB2_INVALID_ARG, "NULL argument");
        fb2_stats_t t{};
        for (auto s : S->ds) {
            t.tokens_generated += s->stats.tokens_generated;
            t.decode_steps += s->stats.decode_steps;
            t.prefill_rows += s->stats.prefill_rows;
            t.reprefills += s->stats.reprefills;
            t.prefill_ms += s->stats.prefill_ms;
            t.decode_ms += s->stats.decode_ms;
            t.sample_ms += s->stats.sample_ms;
            t.kernel_launches += s->stats.kernel_launches;
            t.persistent_steps += s->stats.persistent_steps;
            t.reused_prefix_rows += s->stats.reused_prefix_rows;
        }
        t.device_count = (int)S->ds.size();
        *out = t;
    });
}

int32_t fb2_stats_reset(fb2_session* S) {
    return guarded([&] {
        if (!S) fail(FB2_INVALID_ARG, "NULL argument");
        for (auto s : S->ds) {
            int dc = s->stats.device_count;
            s->stats = fb2_stats_t{};
            s->stats.device_count = dc;
        }
    });
}

// ---- forward_last without allocation --------------------------------------
// ForwardLast of one window through the same prefill kernels as
// fb2_forward_last_logits, with every intermediate (activations, a KV cache
// sized for the window, split-K partial sums and tickets, row tables) in
// g_noalloc_scratch.  No cudaMalloc/cudaFree, no host staging: tokens and
// logits are the caller's device buffers, work is enqueued on the caller's
// stream and the call returns without waiting.
int32_t fb2_forward_last_logits_noalloc(fb2_model* m, int32_t device_slot, int32_t n_tokens,
                                        const int32_t* device_tokens, float* device_logits, void* cuda_stream) {
    return guarded([&] {
        if (!m || !device_tokens || !device_logits) fail(FB2_INVALID_ARG, "NULL argument");
        if (device_slot < 0 || device_slot >= (int)m->devs.size()) fail(FB2_INVALID_ARG, "device slot out of range");
        if (n_tokens < 1) fail(FB2_INVALID_ARG, "Need at least one token.");
        if (n_tokens > kNoallocMaxRows || n_tokens > m->ctx)
            fail(FB2_INVALID_ARG, "fb2_forward_last_logits_noalloc: window of " + std::to_string(n_tokens) +
                                      " tokens exceeds its limit of " + std::to_string(kNoallocMaxRows) +
                                      " (and the context length)");
        const NoallocLayout lay = noalloc_layout(*m);
        if (lay.total > kNoallocScratchFloats)
            fail(FB2_UNSUPPORTED, "fb2_forward_last_logits_noalloc: this model needs " +
                                      std::to_string(lay.total * 4) + " bytes of scratch; the library reserves " +
                                      std::to_string(kNoallocScratchFloats * 4));
        const DeviceModel& dm = m->devs[device_slot];
        // the split-K partial sums of every projection of this window must fit
        // their region, checked before anything is enqueued
        const size_t part_cap = (size_t)512 * 1024;
        const int KN[4][2] = {{m->D, 3 * m->D}, {m->D, m->D}, {m->D, m->F}, {m->F, m->D}};
        for (const auto& kn : KN) {
            const GemvSplit sp = gemv_split(dm.sm_count, kn[0], kn[1]);
            if (sp.S > 1 && (size_t)sp.S * n_tokens * kn[1] > part_cap)
                fail(FB2_UNSUPPORTED, "fb2_forward_last_logits_noalloc: the split-K partial sums of a " +
                                          std::to_string(kn[0]) + "x" + std::to_string(kn[1]) + " projection over " +
                                          std::to_string(n_tokens) + " tokens exceed the scratch region");
        }
        DeviceGuard g(dm.device);
        float* base = nullptr;
        {
            std::lock_guard<std::mutex> lk(g_noalloc_mutex);
            if (dm.device < 0 || dm.device >= 256) fail(FB2_UNSUPPORTED, "device ordinal out of range");
            if (!g_noalloc_ptr[dm.device]) {
                // first call on this device: resolve the array's device address
                // (with this device current)
                CK(cudaGetSymbolAddress((void**)&g_noalloc_ptr[dm.device], g_noalloc_scratch));
            }
            base = g_noalloc_ptr[dm.device];
        }
        // A model view whose context is the window limit: the KV cache in the
        // scratch holds kNoallocMaxRows positions per head.
        fb2_model view;
        view.desc = m->desc;
        view.V = m->V; view.ctx = kNoallocMaxRows; view.D = m->D; view.L = m->L;
        view.H = m->H; view.hd = m->hd; view.F = m->F;
        DeviceSession s;
        s.model = &view;
        s.dm = &dm;
        s.device = dm.device;
        s.nslots = 0;  // head output goes straight to device_logits (row 0)
        s.stream = static_cast<cudaStream_t>(cuda_stream);
        s.d_x = base + lay.x; s.d_x2 = base + lay.x2; s.d_ln = base + lay.ln; s.d_q = base + lay.q;
        s.d_att = base + lay.att; s.d_h = base + lay.h; s.d_lnf = base + lay.lnf;
        s.d_kv = base + lay.kv;
        s.kv_layer_stride = 2LL * view.H * view.ctx * view.hd;
        s.v_offset = (long long)view.H * view.ctx * view.hd;
        s.kv_slot_stride = s.kv_layer_stride * view.L;
        s.d_gemv_part = base + lay.part;
        s.gemv_part_cap = part_cap;
        s.d_tickets = reinterpret_cast<unsigned int*>(base + lay.tickets);
        int* ints = reinterpret_cast<int*>(base + lay.ints);
        s.d_row_hidx = ints + 2 * kNoallocMaxRows;
        s.d_ones = ints + 3 * kNoallocMaxRows;
        s.d_len = ints + 4 * kNoallocMaxRows + 6;
        s.d_hist = const_cast<int*>(device_tokens);
        s.hist_cap = n_tokens;
        s.d_logits = device_logits;
        launch_pdl(k_noalloc_tables, 1, 256, 0, s.stream, n_tokens, ints, s.d_tickets);
        // the prefill chunk of run_prefill_chunk, for this single window
        const int* row_seq = ints;                    // slot 0 for every row
        const int* row_pos = ints + kNoallocMaxRows;  // positions 0..n-1
        const int4* qblk = reinterpret_cast<const int4*>(ints + 4 * kNoallocMaxRows);
        const int* last_row = ints + 4 * kNoallocMaxRows + 4;
        launch_pdl(k_prefill_hidx, 1, 256, 0, s.stream, n_tokens, row_seq, row_pos, s.d_len, view.ctx, s.d_row_hidx);
        Rows R{row_seq, row_pos, s.d_row_hidx, s.d_ones};
        launch_pdl(k_embed, n_tokens, 128, 0, s.stream, n_tokens, R, s.d_hist, s.hist_cap, dm.tok_emb, dm.pos_emb, view.D,
                                                view.V, s.d_x);
        run_layers(s, n_tokens, R, false, QBlocks{1, qblk, 0, nullptr});
        launch_layernorm(s, 1, s.d_x, dm.lnf_w, dm.lnf_b, s.d_lnf, last_row);
        launch_head(s, 1, s.d_lnf, nullptr, device_logits);
        CK(cudaGetLastError());
    });
}

// ---- test hooks (not part of the reference surface) -------------------------
// Copies the persistent kernel's per-phase %globaltimer stamps of its last
// traced launch (FORGE_B200_MK_TRACE=<steps> at session creation) into out:
// [CTAs][steps][64] uint64; *n_ctas / *n_steps receive the shape.
// ---- FORGEMODEL1 ---------------------------------------------------------------
static fb2_model_desc fm_desc(const fb2::fm::Header& h) {
    fb2_model_desc d{};
    d.vocab_size = h.vocab;
    d.context_length = h.ctx;
    d.d_model = h.d_model;
    d.n_layers = h.n_layers;
    d.n_heads = h.n_heads;
    d.weight_dtype = FB2_WEIGHTS_FP32;
    return d;
}

int32_t fb2_forgemodel_read_header(const char* path, fb2_model_desc* out_desc, char* name, int32_t name_capacity) {
    return guarded([&] {
        if (!path || !out_desc) fail(FB2_INVALID_ARG, "NULL argument");
        const fb2::fm::File f = fb2::fm::read_file(path);
        *out_desc = fm_desc(f.hdr);
        if (name && name_capacity > 0) {
            const size_t n = std::min(f.hdr.name.size(), (size_t)name_capacity - 1);
            std::memcpy(name, f.hdr.name.data(), n);
            name[n] = 0;
        }
    });
}

int32_t fb2_model_load_forgemodel(const char* path, int32_t weight_dtype, const int32_t* devices, int32_t n_devices,
                                  fb2_model_desc* out_desc, fb2_model** out) {
    return guarded([&] {
        if (!path || !out) fail(FB2_INVALID_ARG, "NULL argument");
        *out = nullptr;
        fb2::fm::File f = fb2::fm::read_file(path);
        fb2_model_desc d = fm_desc(f.hdr);
        d.weight_dtype = weight_dtype;
        const std::vector<long long> numel = param_numels(d);
        // the weights are 4-byte aligned only if the header length is; copy otherwise
        std::vector<float> aligned;
        const unsigned char* base = f.bytes.data() + f.weights_at;
        const float* w = reinterpret_cast<const float*>(base);
        if (reinterpret_cast<uintptr_t>(base) % alignof(float)) {
            long long total = 0;
            for (long long k : numel) total += k;
            aligned.resize((size_t)total);
            std::memcpy(aligned.data(), base, (size_t)total * 4);
            w = aligned.data();
        }
        std::vector<const float*> ptrs;
        for (long long k : numel) {
            ptrs.push_back(w);
            w += k;
        }
        const int32_t st = fb2_model_create(&d, ptrs.data(), (int32_t)ptrs.size(), devices, n_devices, out);
        if (st != FB2_OK) fail(st, g_last_error);
        if (out_desc) *out_desc = d;
    });
}

int32_t fb2_forgemodel_write(const char* path, const fb2_model_desc* desc, const char* model_name,
                             const float* const* params, int32_t n_params) {
    return guarded([&] {
        if (!path || !desc || !params) fail(FB2_INVALID_ARG, "NULL argument");
        const fb2_model_desc& d = *desc;
        if (d.vocab_size <= 0 || d.context_length <= 0 || d.d_model <= 0 || d.n_layers <= 0 || d.n_heads <= 0 ||
            d.d_model % d.n_heads)
            fail(FB2_INVALID_ARG, "invalid model configuration");
        if (n_params != 4 + 12 * d.n_layers) fail(FB2_INVALID_ARG, "n_params must be 4 + 12*n_layers");
        for (int i = 0; i < n_params; i++)
            if (!params[i]) fail(FB2_INVALID_ARG, "parameter pointer is NULL");
        fb2::fm::Header h;
        h.vocab = d.vocab_size;
        h.ctx = d.context_length;
        h.d_model = d.d_model;
        h.n_layers = d.n_layers;
        h.n_heads = d.n_heads;
        h.name = model_name ? model_name : "";
        bool blank = true;
        for (char c : h.name)
            if (!std::isspace((unsigned char)c)) blank = false;
        if (blank) fail(FB2_INVALID_ARG, "a checkpoint needs a model name");
        fb2::fm::write_file(path, h, params, n_params);
    });
}

// ---- tokenizer ------------------------------------------------------------------
struct fb2_tokenizer {
    fb2::tok::Bpe bpe;
};

int32_t fb2_tokenizer_load(const char* path, fb2_tokenizer** out) {
    return guarded([&] {
        if (!path || !out) fail(FB2_INVALID_ARG, "NULL argument");
        *out = nullptr;
        auto t = std::make_unique<fb2_tokenizer>();
        t->bpe = fb2::tok::Bpe::load(path);
        *out = t.release();
    });
}

void fb2_tokenizer_destroy(fb2_tokenizer* t) { delete t; }

int32_t fb2_tokenizer_info(const fb2_tokenizer* t, int32_t* vocab_size, int32_t* eos_id) {
    return guarded([&] {
        if (!t) fail(FB2_INVALID_ARG, "NULL argument");
        if (vocab_size) *vocab_size = (int32_t)t->bpe.vocab.size();
        if (eos_id) *eos_id = t->bpe.eos;
    });
}

int32_t fb2_tokenizer_encode(const fb2_tokenizer* t, const uint8_t* bytes, int64_t n_bytes, int32_t* ids,
                             int64_t capacity, int64_t* n_ids) {
    return guarded([&] {
        if (!t || !n_ids || (n_bytes > 0 && !bytes) || n_bytes < 0) fail(FB2_INVALID_ARG, "bad arguments");
        const std::vector<int32_t> v = t->bpe.encode(bytes, (size_t)n_bytes);
        *n_ids = (int64_t)v.size();
        if ((int64_t)v.size() > capacity || (!ids && !v.empty())) fail(FB2_INVALID_ARG, "ids buffer too small");
        if (!v.empty()) std::memcpy(ids, v.data(), v.size() * sizeof(int32_t));
    });
}

int32_t fb2_tokenizer_decode(const fb2_tokenizer* t, const int32_t* ids, int64_t n_ids, uint8_t* bytes,
                             int64_t capacity, int64_t* n_bytes) {
    return guarded([&] {
        if (!t || !n_bytes || (n_ids > 0 && !ids) || n_ids < 0) fail(FB2_INVALID_ARG, "bad arguments");
        int64_t total = 0;
        for (int64_t i = 0; i < n_ids; i++) {
            if (ids[i] < 0 || ids[i] >= (int32_t)t->bpe.vocab.size())
                fail(FB2_INVALID_ARG, "token id " + std::to_string(ids[i]) + " is outside the vocabulary");
            total += (int64_t)t->bpe.vocab[(size_t)ids[i]].size();
        }
        *n_bytes = total;
        if (total > capacity || (!bytes && total)) fail(FB2_INVALID_ARG, "bytes buffer too small");
        int64_t at = 0;
        for (int64_t i = 0; i < n_ids; i++) {
            const std::vector<uint8_t>& b = t->bpe.vocab[(size_t)ids[i]];
            if (!b.empty()) std::memcpy(bytes + at, b.data(), b.size());
            at += (int64_t)b.size();
        }
    });
}

int32_t fb2_test_sha256(const void* data, int64_t n, uint8_t* out32) {
    return guarded([&] {
        if ((!data && n) || n < 0 || !out32) fail(FB2_INVALID_ARG, "bad arguments");
        fb2::fm::Sha256 h;
        h.update(data, (size_t)n);
        h.finish(out32);
    });
}

int32_t fb2_test_gemm_tc(int32_t M, int32_t N, int32_t K, const float* A, const float* W, float* out) {
    return guarded([&] {
        if (!A || !W || !out) fail(FB2_INVALID_ARG, "NULL argument");
        if (M <= 0 || N <= 0 || K <= 0 || (N % 4) || (K % 4)) fail(FB2_INVALID_ARG, "bad GEMM shape");
        if (!tc_encode_fn()) fail(FB2_UNSUPPORTED, "cuTensorMapEncodeTiled unavailable");
        int dev = 0;
        CK(cudaGetDevice(&dev));
        configure_kernels(dev);
        const size_t na = (size_t)M * K, nw = (size_t)K * N, no = (size_t)M * N;
        float* buf = dalloc<float>(3 * na + 4 * nw + no + (size_t)N);
        float *a = buf, *ahi = a + na, *alo = ahi + na, *w = alo + na, *whi = w + nw, *wlo = whi + nw, *wt = wlo + nw,
              *o = wt + nw;
        float* bias = o + no;
        int* err = dalloc<int>(1);
        float* part = nullptr;
        try {
            CK(cudaMemcpy(a, A, na * 4, cudaMemcpyHostToDevice));
            CK(cudaMemcpy(w, W, nw * 4, cudaMemcpyHostToDevice));
            CK(cudaMemset(bias, 0, (size_t)N * 4));
            CK(cudaMemset(err, 0, sizeof(int)));
            launch_split_tf32_transpose(0, w, K, N, whi, wlo, wt);
            CUtensorMap bm[3];
            if (!tc_encode(&bm[0], whi, K, N, 128) || !tc_encode(&bm[1], wlo, K, N, 128) ||
                !tc_encode(&bm[2], wt, K, N, 128))
                fail(FB2_CUDA_ERROR, "cuTensorMapEncodeTiled failed");
            const size_t cap = (size_t)kTcSplitMax * M * N;
            part = dalloc<float>(cap);
            int64_t launches = 0;
            Epi e = make_epi(EPI_BIAS, bias, nullptr, o);
            if (!launch_gemm_tc(0, 148, M, K, N, a, ahi, alo, bm, e, err, part, cap, &launches, false))
                fail(FB2_UNSUPPORTED, "the tensor-core GEMM takes more than 16 rows");
            CK(cudaGetLastError());
            CK(cudaDeviceSynchronize());
            int herr = 0;
            CK(cudaMemcpy(&herr, err, sizeof(int), cudaMemcpyDeviceToHost));
            if (herr) fail(FB2_TIMEOUT, "tensor-core GEMM: a bounded wait expired");
            CK(cudaMemcpy(out, o, no * 4, cudaMemcpyDeviceToHost));
        } catch (...) {
            dfree(buf);
            dfree(err);
            dfree(part);
            throw;
        }
        dfree(buf);
        dfree(err);
        dfree(part);
    });
}

int32_t fb2_test_mk_trace(fb2_session* S, uint64_t* out, int64_t capacity, int32_t* n_ctas, int32_t* n_steps) {
    return guarded([&] {
        if (!S || !n_ctas || !n_steps) fail(FB2_INVALID_ARG, "NULL argument");
        DeviceSession& s = *S->ds[0];
        *n_ctas = s.mk_trace ? s.dm->mk_nW : 0;
        *n_steps = s.mk_trace ? s.mk_trace_steps : 0;
        if (!s.mk_trace || !out) return;
        const size_t n = (size_t)s.dm->mk_nW * s.mk_trace_steps * MK_TRACE_POINTS;
        if ((size_t)capacity < n) fail(FB2_INVALID_ARG, "capacity too small");
        DeviceGuard g(s.device);
        CK(cudaStreamSynchronize(s.stream));
        CK(cudaMemcpy(out, s.mk_trace, n * 8, cudaMemcpyDeviceToHost));
    });
}

// n successive NextDouble() values of `new Random(seed)` as the library
// restates it (host code; needs no device).
int32_t fb2_test_mk_withhold(fb2_session* S, int32_t cta, int64_t wait_ns) {
    return guarded([&] {
        if (!S || S->ds.empty()) fail(FB2_INVALID_ARG, "session is NULL");
        if (cta < 0 || wait_ns <= 0 || wait_ns > (int64_t)MK_TIMEOUT_NS) fail(FB2_INVALID_ARG, "bad hook arguments");
        DeviceSession& s = *S->ds[0];
        if (!s.mk_use) fail(FB2_UNSUPPORTED, "the session does not use the persistent decode kernel");
        if (cta >= s.dm->mk_nW) fail(FB2_INVALID_ARG, "no such CTA");
        s.test_withhold_cta = cta;
        s.test_wait_ns = (unsigned long long)wait_ns;
    });
}

int32_t fb2_test_mk_geometry(fb2_session* S, int32_t* n_ctas, int32_t* cluster, int32_t* attn_ctas, int32_t* stages) {
    return guarded([&] {
        if (!S || S->ds.empty() || !n_ctas || !cluster || !attn_ctas || !stages) fail(FB2_INVALID_ARG, "NULL argument");
        DeviceSession& s = *S->ds[0];
        const DeviceModel& dm = *s.dm;
        *n_ctas = s.mk_use ? dm.mk_nW : 0;
        *cluster = dm.mk_hc ? dm.mk_cs : 0;
        *attn_ctas = dm.mk_hc ? dm.mk_nhead : 0;
        int ns = s.mk_use ? mk_nstage(*s.model, 1, dm.mk_nW, s.device, dm.mk_hc ? dm.mk_cs : 0) : 0;
        if (s.mk_use && dm.mk_hc) {
            const int n32 = mk_nstage(*s.model, 1, dm.mk_nW, s.device, dm.mk_cs, MK_STAGE_HC);
            if (n32 >= 5) ns = n32;  // 32 KB stages
        }
        *stages = ns;
    });
}

int32_t fb2_test_fail_alloc(int64_t nth, int64_t* allocs_so_far) {
    return guarded([&] {
        if (nth < 0) fail(FB2_INVALID_ARG, "nth must be >= 0");
        if (allocs_so_far) *allocs_so_far = g_alloc_count.load();
        g_fail_alloc_at = nth > 0 ? g_alloc_count.load() + nth : 0;
    });
}

int32_t fb2_test_dotnet_random(int32_t seed, int32_t n, double* out) {
    return guarded([&] {
        if (!out || n < 0) fail(FB2_INVALID_ARG, "bad arguments");
        DotNetRandom r(seed);
        for (int i = 0; i < n; i++) out[i] = r.next_double();
    });
}

// Device expf_libm over n inputs (host arrays).
int32_t fb2_test_expf(const float* x, float* y, int64_t n) {
    return guarded([&] {
        if (!x || !y || n <= 0) fail(FB2_INVALID_ARG, "bad arguments");
        float *dx = dalloc<float>(n), *dy = dalloc<float>(n);
        CK(cudaMemcpy(dx, x, n * 4, cudaMemcpyHostToDevice));
        k_expf_libm<<<ceil_div(n, 256), 256>>>(dx, dy, n);
        cudaError_t e = cudaGetLastError();
        if (e == cudaSuccess) e = cudaMemcpy(y, dy, n * 4, cudaMemcpyDeviceToHost);
        cudaFree(dx);
        cudaFree(dy);
        CK(e);
    });
}

// Per-chunk (2^20 inputs) hashes of expf_libm over [lo_bits, lo_bits + nchunks*2^20).
int32_t fb2_test_expf_hash(uint32_t lo_bits, int32_t nchunks, uint64_t* hashes) {
    return guarded([&] {
        if (!hashes || nchunks <= 0) fail(FB2_INVALID_ARG, "bad arguments");
        unsigned long long* d = dalloc<unsigned long long>(nchunks);
        CK(cudaMemset(d, 0, nchunks * 8));
        k_expf_libm_hash<<<nchunks, 1024>>>(lo_bits, nchunks, d);
        cudaError_t e = cudaGetLastError();
        if (e == cudaSuccess) e = cudaMemcpy(hashes, d, nchunks * 8, cudaMemcpyDeviceToHost);
        cudaFree(d);
        CK(e);
    });
}

}  // extern "C"
