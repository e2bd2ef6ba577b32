from ue5m3_fp4.nn.convert import (ConversionRecord, ProductPlan, convert_linear_modules, exclude_lm_head,
                                  plan_fp4_products, reserve_device_workspace, select_all_linears)
from ue5m3_fp4.nn.linear import LinearBackend, UE5M3Linear
from ue5m3_fp4.nn.packed_linear import PackedFP4Linear, pack_frozen_linears

__all__ = [
    "ConversionRecord",
    "LinearBackend",
    "PackedFP4Linear",
    "ProductPlan",
    "UE5M3Linear",
    "plan_fp4_products",
    "reserve_device_workspace",
    "convert_linear_modules",
    "exclude_lm_head",
    "pack_frozen_linears",
    "select_all_linears",
]
