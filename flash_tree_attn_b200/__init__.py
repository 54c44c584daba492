"""B200-native tree-attention decode: a drop-in for `flash_tree_attn.flash_decoding_attention`.

    from flash_tree_attn_b200 import flash_decoding_attention

Beside it the other operators of a decoding loop: `decode_attention(_paged)`, `append_tokens`, `apply_rotary`,
`evict_rows`, `commit_accepted`, `token_logprobs`, and a layer that uses them, `TreeVerifyAttention`.

The arithmetic lives in libfta.so (hand-written sm_100a CUDA behind the C ABI of
include/fta.h); build it with `python -m flash_tree_attn_b200.build`.
"""
from .op import (  # noqa: F401
    check_status,
    commit_accepted,
    flash_decoding_attention,
    flash_decoding_attention_paged,
    flash_decoding_attention_with_lse,
    merge_partials,
    prepare,
    set_grid_override,
    set_kernel,
    set_split_mode,
)

from .decode import decode_attention, decode_attention_paged, evict_rows  # noqa: F401,E402
from .logprobs import TokenLogprobs, token_logprobs  # noqa: F401,E402
from .rotary import append_tokens, apply_rotary, rotary_frequencies  # noqa: F401,E402
from .speculative import (  # noqa: F401,E402
    DraftTree,
    TreeVerifyAttention,
    accept_longest_path,
    greedy_node_ok,
    typical_node_ok,
)

__all__ = [
    "check_status",
    "DraftTree",
    "TreeVerifyAttention",
    "accept_longest_path",
    "append_tokens",
    "apply_rotary",
    "commit_accepted",
    "decode_attention",
    "decode_attention_paged",
    "evict_rows",
    "flash_decoding_attention",
    "flash_decoding_attention_paged",
    "flash_decoding_attention_with_lse",
    "greedy_node_ok",
    "merge_partials",
    "prepare",
    "rotary_frequencies",
    "set_split_mode",
    "set_kernel",
    "set_grid_override",
    "token_logprobs",
    "TokenLogprobs",
    "typical_node_ok",
]
