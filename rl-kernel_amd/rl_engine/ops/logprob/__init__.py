"""Selected-token log-probability operators (the reference leaves this package
as an empty extension point, rl_engine/ops/logprob/__init__.py)."""

from rl_engine.backends.rocm.logprob.token_scores import (
    TokenScores,
    hip_deterministic_linear_scores as deterministic_linear_scores,
    hip_deterministic_scores_from_logits as deterministic_scores_from_logits,
)
from rl_engine.backends.rocm.logprob.vocab_parallel_logp import (
    RocmVocabParallelLogprobOp as VocabParallelLogprobOp,
    hip_deterministic_logp_from_logits as deterministic_logp_from_logits,
    merge_tile_partials,
)
from rl_engine.ops.logprob.linear_logp import (
    LinearLogpOp,
    deterministic_linear_logp,
    linear_logp,
    linear_logp_contract_version,
    recompute_logits,
)

__all__ = [
    "LinearLogpOp",
    "TokenScores",
    "VocabParallelLogprobOp",
    "deterministic_linear_logp",
    "deterministic_linear_scores",
    "deterministic_logp_from_logits",
    "deterministic_scores_from_logits",
    "linear_logp",
    "linear_logp_contract_version",
    "merge_tile_partials",
    "recompute_logits",
]
