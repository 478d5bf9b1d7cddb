"""Tree acceptance and KV compaction (drop-in for ``diffspec.draft.tree_verification``)."""

from .tree_verification import (AcceptResult, accept, accept_residual, compact_kv, prepare_logits_processor, verify,
                                verify_new)

__all__ = ["AcceptResult", "accept", "accept_residual", "compact_kv", "prepare_logits_processor", "verify", "verify_new"]
