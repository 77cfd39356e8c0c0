"""nvjsel -- MI355X-native decode-step token selection (LM-head top-1 + sampler).

Import with ``nano-vllm-jax_amd`` on ``sys.path`` (the repo-root entry points
and tests do this).  The compute lives in ``libnvjsel.so`` (HIP, gfx950); see
``include/nvjsel.h`` for the C ABI.
"""
from ._lib import NativeLibraryMissing, NvjselError, load
from .adapters import AdapterTable, apply_adapters, pack_adapters
from .beam import beam_search_select, lm_head_beam_search_step, reorder_beam_states
from .logprobs import TokenLogprobs, lm_head_token_logprobs, token_logprobs
from .registry import (
    KernelBackendUnavailable,
    available_backends,
    lm_head_greedy_top1_impl,
    mtp_lm_head_greedy_top1_impl,
    select_token_selection_backend,
)
from .selection import (
    derive_rng_keys,
    derive_rng_keys_from_table,
    lm_head_greedy_top1_hip,
    lm_head_logits_hip,
    lm_head_sample_token_ids,
    lm_head_token_ids_and_topk,
    mtp_greedy_top1_token_ids,
    reference_reduce_cast,
    reset_rng_counters,
    rms_norm_hip,
    sample_token_ids,
    topk_hip,
)
from .w4 import W4Weight, pack_lm_head_w4, quantize_lm_head_w4

__all__ = [
    "AdapterTable",
    "NativeLibraryMissing",
    "NvjselError",
    "KernelBackendUnavailable",
    "TokenLogprobs",
    "W4Weight",
    "apply_adapters",
    "available_backends",
    "beam_search_select",
    "derive_rng_keys",
    "derive_rng_keys_from_table",
    "load",
    "lm_head_beam_search_step",
    "lm_head_greedy_top1_hip",
    "lm_head_greedy_top1_impl",
    "lm_head_logits_hip",
    "lm_head_sample_token_ids",
    "lm_head_token_ids_and_topk",
    "lm_head_token_logprobs",
    "mtp_greedy_top1_token_ids",
    "mtp_lm_head_greedy_top1_impl",
    "pack_adapters",
    "pack_lm_head_w4",
    "quantize_lm_head_w4",
    "reference_reduce_cast",
    "reorder_beam_states",
    "reset_rng_counters",
    "rms_norm_hip",
    "sample_token_ids",
    "select_token_selection_backend",
    "token_logprobs",
    "topk_hip",
]
