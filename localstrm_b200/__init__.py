"""B200-native (sm_100a) batched token sampler with LocalStrm's sampling semantics.

The hot path is one native library (``_lib/liblss.so``, built from ``csrc/``) behind the
C ABI in ``include/lsampler.h``; ``sampling`` is the drop-in for the reference's
``src/engine/sampling.py`` and ``distributed`` holds the row- and vocabulary-sharded modes.
``head`` (the 4-bit vocabulary projection) and ``paged`` (block tables, the 8-bit key/value cache
and its attention) are the rest of the decode step around it, with ``rotary`` (norms and position
rotation of queries and keys) and ``drafts`` (trees of drafted tokens and their acceptance).
"""
from .head import Int4Weight, int4_matvec, sample_hidden  # noqa: F401
from .drafts import Accepted, accept_drafts, compact_kv, plan_tree  # noqa: F401
from .paged import (Forks, KVCache8, StepPlan, TreePlan, append_kv, attend, copy_blocks, fork_blocks,  # noqa: F401
                    plan_blocks, release_blocks)
from .rotary import norm_rotate  # noqa: F401
from .sampling import (BatchSampler, RowParams, SamplerError, SamplingParams,  # noqa: F401
                       STOP_EOS, STOP_NONE, STOP_TOKEN, apply_top_k_top_p_min_p, check_stop_batch,
                       greedy_batch, sample_batch, sample_next_token, stop_reasons)

__version__ = "0.1.0"
