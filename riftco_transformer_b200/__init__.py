"""B200 (sm_100a) backend for Riftco's packed-NF4 linear and paged-KV decode
attention. The product is the CUDA library behind ``include/riftco_b200.h``;
this package is its host-side face for Python callers, shaped after the
reference's backend operator interface.

Attributes are resolved on first use so that ``python -m
riftco_transformer_b200.build`` can run before the shared library exists.
"""
_EXPORTS = (
    "DomainError",
    "BackendUnavailable",
    "PackedNf4Weight",
    "PagedKvPool",
    "PagedKv4Pool",
    "check_device_errors",
    "dequantize",
    "dequantize_kv4",
    "dispatch_paged_decode_attention_forward",
    "dispatch_quantized_linear_forward",
    "dispatch_quantized_linear_input_backward",
    "host_paged_decode_attention_forward",
    "host_quantized_linear_forward",
    "host_quantized_linear_input_backward",
    "is_available",
    "last_route",
    "paged_chunk_attention_kv4",
    "paged_chunk_kv4_workspace_bytes",
    "paged_decode_attention",
    "paged_decode_attention_kv4",
    "paged_decode_kv4_workspace_bytes",
    "quantize_nf4",
    "rope_append_kv4",
    "unavailability_reason",
    "validate_payload",
)
__all__ = list(_EXPORTS)


def __getattr__(name):
    if name in _EXPORTS:
        from . import backend, kv4
        value = getattr(kv4 if name in kv4.__all__ else backend, name)
        globals()[name] = value   # later uses are plain attributes
        return value
    raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
