"""turbopress_amd: TurboPress's packed-TCQ decode path, native to MI355X (gfx950).

Drop-in for the reference's packed runtime (turbopress/runtime.py,
turbopress/triton_kernel.py): ``PackedTCQLinear`` takes the same format-v2
payload and forward signature; ``fwht_scale``/``packed_gemv`` keep the
reference kernel wrappers' names.  All compute runs in hand-written HIP
kernels from ``libturbopress_amd.so`` (C ABI in ``include/turbopress_amd.h``).
"""

from __future__ import annotations

__version__ = "0.1.0"

_LAZY = {
    "PackedTCQLinear": ("turbopress_amd.runtime", "PackedTCQLinear"),
    "Trellis": ("turbopress_amd.runtime", "Trellis"),
    "HAS_HIP": ("turbopress_amd.hip_kernel", "HAS_HIP"),
    "fwht_scale": ("turbopress_amd.hip_kernel", "fwht_scale"),
    "packed_gemv": ("turbopress_amd.hip_kernel", "packed_gemv"),
    "subset_lut": ("turbopress_amd.hip_kernel", "subset_lut"),
    "window_decode_levels": ("turbopress_amd.hip_kernel", "window_decode_levels"),
    "default_codebook": ("turbopress_amd.codebooks", "default_codebook"),
    "pack_linear": ("turbopress_amd.pack", "pack_linear"),
    "pack_model": ("turbopress_amd.pack", "pack_model"),
    "load_packed_model": ("turbopress_amd.artifact", "load_packed_model"),
    "tcq_quantize_rows": ("turbopress_amd.encoder", "tcq_quantize_rows"),
    "rms_norm": ("turbopress_amd.norm", "rms_norm"),
    "rms_norm_fp8": ("turbopress_amd.norm", "rms_norm_fp8"),
    "fp8_linear": ("turbopress_amd.fp8", "fp8_linear"),
    "quantize_fp8_weight": ("turbopress_amd.fp8", "quantize_fp8_weight"),
    "rotary_table": ("turbopress_amd.paged", "rotary_table"),
    "rotary": ("turbopress_amd.paged", "rotary"),
    "rotary_append": ("turbopress_amd.paged", "rotary_append"),
    "paged_attention": ("turbopress_amd.paged", "paged_attention"),
    "paged_tree_attention": ("turbopress_amd.paged", "paged_tree_attention"),
    "tree_ancestors": ("turbopress_amd.paged", "tree_ancestors"),
    "token_logprobs": ("turbopress_amd.logprobs", "token_logprobs"),
    "lora_add": ("turbopress_amd.lora", "lora_add"),
    "LoraAdapters": ("turbopress_amd.lora", "LoraAdapters"),
    "PagedDecoder": ("turbopress_amd.paged_decode", "PagedDecoder"),
}

__all__ = list(_LAZY)


def __getattr__(name):
    if name in _LAZY:
        import importlib
        mod, attr = _LAZY[name]
        value = globals()[name] = getattr(importlib.import_module(mod), attr)
        return value  # (found without this function from now on: it took 3 us per use)
    raise AttributeError(f"module 'turbopress_amd' has no attribute {name!r}")
