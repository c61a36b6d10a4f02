"""Re-exports of the hot-path kernels (reference forge/forge/kernels/__init__.py):

    forge.kernels.swiglu         ForgeSwiGLUFunction, swiglu, ...  (kernels/swiglu)
    forge.kernels.geglu          ForgeGEGLUFunction, geglu, ...    (kernels/geglu)
    forge.kernels.rope           apply_rope, ForgeRoPEv3, forge_apply_rotary_pos_emb
                                 apply_qk_norm_rope (q/k norms and RoPE in one pass)
    forge.kernels.glu_act8       glu_act8, glu_act8_packed (gate and up kept in 8 bits)
    forge.kernels.logprob        forge_token_logps, forge_preference_loss, forge_policy_loss
    forge.kernels.cross_entropy  ForgeCrossEntropyFunction, forge_cross_entropy,
                                 ForgeFusedLinearCrossEntropyFunction, ...
    forge.kernels.lora_mlp       LoRAMLPv3 / LoRAMLPv6 and helpers
    forge.kernels.lora_qkv       LoRAQKVFunction / LoRAQKVv4Function and helpers
"""
