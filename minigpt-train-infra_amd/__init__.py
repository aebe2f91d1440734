"""MI355X-native optimizer step for MiniGPT-style training.

Drop-in replacements for the torch calls of the reference's training loop
(train.py:359-370, 457-491):

    AdamW            for torch.optim.AdamW
    GradScaler       for torch.amp.GradScaler
    clip_grad_norm_  for torch.nn.utils.clip_grad_norm_

plus the loop's host helpers (build_adamw_param_groups, set_optimizer_lr,
cosine_lr, optimizer_completed_steps) and the checkpoint loaders it calls on
resume (load_optimizer_state, load_grad_scaler_state).  Beside them, the
operators of a training step around its matrix products, and of a rollout:

    embedding       lookup of scaled rows, and the weight's gradient
    add_rms_norm    the residual's addition and the RMS norm of the sum
    qk_norm_rope    RMS norms of query and key heads and the rotary rotation
    attention       grouped heads over batches, packed sequences and caches
    int8_linear     products of 8-bit integers with scales per token and channel
    gated_act       the MLP's activation with an 8-bit checkpoint
    policy_loss     the clipped policy loss with a KL term over the logits

The arithmetic runs
in hand-written gfx950 kernels (libmgopt.so, C ABI in include/mgopt.h); there
is no CPU path.

The package directory name contains hyphens, so import it with
importlib.import_module("minigpt-train-infra_amd").
"""

from .adamw import AdamW
from .attention import attention, attention_backward, attention_lse
from .clip_grad import clip_grad_norm_
from .embedding import embedding, embedding_grad_
from .gated_act import ActCheckpoint, gated_act, gated_act_backward, gated_act_pack
from .grad_scaler import GradScaler
from .int8_linear import Int8Rows, int8_linear, int8_rows
from .policy_loss import PolicyLoss, policy_loss, policy_loss_grad, token_log_probs
from .qk_norm_rope import qk_norm_rope, qk_norm_rope_backward, rope_tables
from .rms_norm import add_rms_norm, rms_norm, rms_norm_backward, rms_norm_int8
from .schedule import build_adamw_param_groups, cosine_lr, optimizer_completed_steps, set_optimizer_lr
from .state_load import load_grad_scaler_state, load_optimizer_state
from . import paramsets

__all__ = [
    "AdamW",
    "GradScaler",
    "clip_grad_norm_",
    "build_adamw_param_groups",
    "cosine_lr",
    "set_optimizer_lr",
    "optimizer_completed_steps",
    "load_optimizer_state",
    "load_grad_scaler_state",
    "paramsets",
    "embedding",
    "embedding_grad_",
    "ActCheckpoint",
    "gated_act",
    "gated_act_backward",
    "gated_act_pack",
    "PolicyLoss",
    "policy_loss",
    "policy_loss_grad",
    "qk_norm_rope",
    "qk_norm_rope_backward",
    "rope_tables",
    "token_log_probs",
    "attention",
    "attention_backward",
    "attention_lse",
    "add_rms_norm",
    "rms_norm",
    "rms_norm_backward",
    "rms_norm_int8",
    "Int8Rows",
    "int8_linear",
    "int8_rows",
]
