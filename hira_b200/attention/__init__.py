from .hira_attention import (HiraDecodeStep, hira_attention, hira_decode_attention, make_hira_attention,
                             register_hira_attention)
from .rope import hira_attention_forward, hira_qk_norm_rope, patch_attention
from .shared_attention import SharedPrompt, hira_shared_attention

__all__ = ["HiraDecodeStep", "hira_attention", "hira_decode_attention", "make_hira_attention", "register_hira_attention",
           "hira_attention_forward", "hira_qk_norm_rope", "patch_attention", "SharedPrompt", "hira_shared_attention"]
