// C ABI of the verification of drafted tokens (include/rl_drafts.h); the kernels are in
// drafts.h.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <new>
#include <string>

#include "drafts.h"
#include "rl_runtime.h"

using namespace rl;

struct rl_drafts {
    int device = 0;
    uint32_t max_seqs = 0, vocab = 0, chunks = 0;
    double *sums = nullptr;
    uint32_t *arrived = nullptr;
    ~rl_drafts() {
        (void)hipFree(sums);
        (void)hipFree(arrived);
    }
};

namespace {

// Workgroups that the chunks of a call are shared among: each finds the accepted drafts first, so few do that more seldom,
// but they have to fill the device. 64 sequences of 61 chunks, us: 512 27.7, 1024 28.2, 2048 51.5.
constexpr uint32_t DRAFT_FILL = 1024;

// What is wrong with a call's probabilities, or null.
const char *wrong(const rl_probs *p, uint32_t vocab) {
    if (!p->probs) return "has no probabilities";
    if ((uintptr_t)p->probs % 4 || (uintptr_t)p->ids % 4 || (uintptr_t)p->kept % 4) return "is not aligned to its type";
    if (!p->ids != !p->kept) return "has ids or kept counts without the others";
    if (!p->ids && p->row_stride < vocab) return "has rows that overlap";
    if (p->ids && p->row_stride == 0) return "has lists without room";
    return nullptr;
}

bool wide(const rl_probs &p) { return !p.probs || ((uintptr_t)p.probs % 16 == 0 && p.row_stride % 4 == 0); }

}  // namespace

extern "C" {

int rl_drafts_create(int device, uint32_t max_seqs, uint32_t vocab, rl_drafts **out) {
    if (!out) return fail(RL_ERR_ARGUMENT, "out is null");
    *out = nullptr;
    if (max_seqs == 0 || vocab == 0) return fail(RL_ERR_ARGUMENT, "max_seqs and vocab must be positive");
    if (max_seqs > 1u << 16 || vocab > 1u << 21) return fail(RL_ERR_CAPACITY, "max_seqs above 2^16 or vocab above 2^21");
    DeviceGuard guard(device);
    if (!guard.ok) return fail(RL_ERR_DEVICE, "cannot select device " + std::to_string(device));
    auto *h = new (std::nothrow) rl_drafts();
    if (!h) return fail(RL_ERR_CAPACITY, "out of host memory");
    h->device = device;
    h->max_seqs = max_seqs, h->vocab = vocab;
    h->chunks = (vocab + DRAFT_CHUNK - 1) / DRAFT_CHUNK;
    hipError_t e = hipMalloc(&h->sums, (size_t)max_seqs * h->chunks * sizeof(double));
    if (e == hipSuccess) e = hipMalloc(&h->arrived, (size_t)max_seqs * sizeof(uint32_t));
    if (e == hipSuccess) e = hipMemset(h->arrived, 0, (size_t)max_seqs * sizeof(uint32_t));
    if (e == hipSuccess) e = hipDeviceSynchronize();
    if (e != hipSuccess) {
        delete h;
        return hip_fail(e, "rl_drafts_create");
    }
    *out = h;
    return RL_OK;
}

void rl_drafts_destroy(rl_drafts *drafts) {
    if (!drafts) return;
    DeviceGuard guard(drafts->device);
    delete drafts;
}

int rl_drafts_verify(rl_drafts *h, const rl_probs *target, const rl_probs *draft, const int32_t *drafted,
                     const int32_t *starts, const float *uniforms, const float *draws, uint32_t drafts, uint32_t seqs,
                     int32_t *accepted, int32_t *tokens, void *stream) {
    if (!h) return fail(RL_ERR_ARGUMENT, "drafts is null");
    if (seqs == 0) return drafts ? fail(RL_ERR_ARGUMENT, "drafts without a sequence") : RL_OK;
    if (!target) return fail(RL_ERR_ARGUMENT, "target is null");
    if (const char *w = wrong(target, h->vocab)) return fail(RL_ERR_ARGUMENT, std::string("target ") + w);
    if (draft && drafts) {
        if (const char *w = wrong(draft, h->vocab)) return fail(RL_ERR_ARGUMENT, std::string("draft ") + w);
        if (!draft->ids != !target->ids) return fail(RL_ERR_ARGUMENT, "target and draft are both lists, or neither");
    }
    if (seqs > h->max_seqs) return fail(RL_ERR_CAPACITY, "seqs above the handle's max_seqs");
    if (drafts > 1u << 23) return fail(RL_ERR_CAPACITY, "more than 2^23 drafts in a call");
    if (!starts || !draws || !accepted || !tokens || (drafts && (!drafted || !uniforms)))
        return fail(RL_ERR_ARGUMENT, "drafted, starts, uniforms, draws, accepted and tokens must be device pointers");
    // Chunks a workgroup: it has to find the row first, which several share, but few sequences want many workgroups.
    const uint32_t per = (uint32_t)std::min<uint64_t>(std::max<uint64_t>((uint64_t)seqs * h->chunks / DRAFT_FILL, 1), DRAFT_PER);
    const uint32_t groups = (h->chunks + per - 1) / per; // times 2^16 sequences: 2^22 workgroups at most
    DeviceGuard guard(h->device);
    if (!guard.ok) return fail(RL_ERR_DEVICE, "cannot select the handle's device");
    DraftArgs a{};
    a.target = *target;
    if (draft && drafts) a.draft = *draft;
    a.drafted = drafted, a.starts = starts, a.uniforms = uniforms, a.draws = draws;
    a.accepted = accepted, a.tokens = tokens;
    a.vocab = h->vocab, a.drafts = drafts, a.seqs = seqs, a.chunks = h->chunks, a.per = per, a.groups = groups;
    a.sums = h->sums, a.arrived = h->arrived;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (target->ids) hipLaunchKernelGGL(k_drafts_lists, dim3(seqs), dim3(DRAFT_THREADS), 0, s, a);
    else if (wide(a.target) && wide(a.draft)) hipLaunchKernelGGL(k_drafts<true>, dim3(seqs * groups), dim3(DRAFT_THREADS), 0, s, a);
    else hipLaunchKernelGGL(k_drafts<false>, dim3(seqs * groups), dim3(DRAFT_THREADS), 0, s, a);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? RL_OK : hip_fail(e, "rl_drafts_verify launch");
}

}  // extern "C"
