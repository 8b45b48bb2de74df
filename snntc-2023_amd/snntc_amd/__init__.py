"""MI355X (gfx950) implementation of the SNN-TC custom ops behind the reference's Python API.

Public names follow the reference module ``SNN_TC_Modules``: the op handles ``snnfc``,
``snnfc_grad``, ``snncv``, ``snncv_grad`` and the layers ``SNN_dense``, ``SNN_conv``,
``SNN_maxpool2d``, ``SNN_avgpool2d``, ``SNN_LRN``, plus ``init_weight`` and ``loss_func``.  For networks over sequences
of tokens: ``SNN_embedding``, ``SNN_recurrence``, ``SNN_steps``, ``policy_loss`` and ``preference_loss`` with their ops.
"""
from . import _lib
from ._lib import SnntcError, SnntcLibraryError
from .ops import SnnCv, SnnCvSame, SnnCvTimes, SnnFc, SnnFcTimes, SnnMinPool, SnnPadTime, SoftmaxTimeLoss, min_pool, min_pool_grad, pad_time, pad_time_grad, sgd_update, softmax_time_loss, snncv, snncv_grad, snncv_output_dims, snnfc, snnfc_grad, snnfc_static, init, check_scan_health
from .ops import (PolicyTimeLoss, PreferenceTimeLoss, SnnEmbed, SnnGatedScan, embed_tokens, embed_tokens_grad, gated_scan, gated_scan_grad,
                  gated_step, policy_time_loss, preference_time_loss, time_logp)
from .ops import TimeRules, adamw_moments, adamw_update, choose_tokens, grad_norm, pack_allowed, rule_times, rule_times_grad
from . import train
from . import optim
from . import networks
from .layers import (SNN_LRN, SNN_avgpool2d, SNN_conv, SNN_dense, SNN_embedding, SNN_flatten, SNN_globalminpool2d, SNN_maxpool2d,
                     SNN_recurrence, SNN_steps, init_weight, loss_func, policy_loss, preference_loss)

__all__ = [
    "snnfc", "snnfc_grad", "snnfc_static", "init", "check_scan_health", "snncv", "snncv_grad", "snncv_output_dims", "SnnFc", "SnnCv", "SnnFcTimes", "SnnCvTimes", "SoftmaxTimeLoss", "softmax_time_loss", "sgd_update", "SnnMinPool", "min_pool", "min_pool_grad", "SnnPadTime", "pad_time", "pad_time_grad",
    "SNN_dense", "SNN_conv", "SNN_maxpool2d", "SNN_avgpool2d", "SNN_globalminpool2d", "SNN_flatten", "SNN_LRN", "init_weight", "loss_func",
    "SnnEmbed", "embed_tokens", "embed_tokens_grad", "SnnGatedScan", "gated_scan", "gated_scan_grad", "gated_step", "time_logp",
    "PolicyTimeLoss", "policy_time_loss", "PreferenceTimeLoss", "preference_time_loss",
    "TimeRules", "rule_times", "rule_times_grad", "choose_tokens", "pack_allowed", "grad_norm", "adamw_update", "adamw_moments",
    "SNN_embedding", "SNN_recurrence", "SNN_steps", "policy_loss", "preference_loss",
    "SnntcError", "SnntcLibraryError", "train", "networks", "optim",
]
