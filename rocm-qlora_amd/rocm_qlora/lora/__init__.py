"""LoRA adapter layers: one adapter (lora/__init__.py of the reference), and
many adapters beside one projection."""
from rocm_qlora.lora.lora_layer import LoRALinear
from rocm_qlora.lora.adapters import AdapterRows, MultiLoRALinear, attach_adapters, multi_lora, set_adapter_rows

__all__ = ["LoRALinear", "AdapterRows", "MultiLoRALinear", "attach_adapters", "multi_lora", "set_adapter_rows"]
