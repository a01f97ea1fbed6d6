"""tabby_b200: B200-native (sm_100a) token sampler, a drop-in for the GPU sampling path
of xOAviOx/tabby (src/engine/sampler.ts + the reduce_max / reduce_sumexp / topk_partial /
topk_select kernels driven by src/engine/forward.ts:520-601), and the decode step over
several hypotheses a sequence next to it: beam search and drafted trees (decode.py)."""
from .sampler import (  # noqa: F401
    DEFAULT_SAMPLING,
    MAX_TOP_K,
    SampleBatch,
    SampleOutcome,
    Sampler,
    SamplingParams,
    SeededRandom,
    TopKResult,
    decode_sample_block,
    pool_size,
    sampleFromTopK,
    sample_from_topk,
)

_DECODE = ("BeamStep", "TreeAccept", "beam_step", "reorder_states", "tree_accept",
           "tree_attention")


def __getattr__(name):  # decode.py imports torch; the sampler's host half does without
    if name in _DECODE:
        from . import decode

        return getattr(decode, name)
    raise AttributeError(f"module {__name__!r} has no attribute {name!r}")


def __dir__():
    return sorted([*globals(), *_DECODE])
