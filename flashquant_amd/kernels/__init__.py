"""Operator layer with the signatures of the reference's ``flashquant.kernels``
(src/flashquant/kernels/__init__.py): tq4_compress, tq4_decompress,
fused_tq_attention, split_k_paged_decode; and operators around a 16-bit paged
cache that the reference takes from elsewhere.  Every call goes to the HIP kernels
through ``flashquant_amd._C``; nothing here computes on the CPU."""
from flashquant_amd.kernels.attention import fused_tq_attention, paged_tq4_prefill
from flashquant_amd.kernels.compress import tq4_compress, tq4_compress_and_store
from flashquant_amd.kernels.decompress import tq4_decompress, tq4_decompress_rotated
from flashquant_amd.kernels.packing import nibble_pack, nibble_unpack, pack_2bit, unpack_2bit
from flashquant_amd.kernels.paged_decode import split_k_paged_decode, tq4_store_and_decode
from flashquant_amd.kernels.paged_kv import PagedSchedule, paged_kv_decode, paged_schedule
from flashquant_amd.kernels.paged_kv8 import paged_kv8_decode, paged_kv8_read, rotary_paged_store8
from flashquant_amd.kernels.paged_prefix import paged_prefix_decode
from flashquant_amd.kernels.prod import prod_compress, prod_paged_decode, prod_page_layout, prod_store_rows
from flashquant_amd.kernels.rotary import rotary_embedding, rotary_frequencies, rotary_paged_store

__all__ = ["tq4_compress", "tq4_compress_and_store", "tq4_decompress", "tq4_decompress_rotated", "fused_tq_attention", "paged_tq4_prefill", "split_k_paged_decode", "tq4_store_and_decode", "nibble_pack", "nibble_unpack", "pack_2bit", "unpack_2bit",
           "prod_compress", "prod_paged_decode", "prod_page_layout", "prod_store_rows", "PagedSchedule", "paged_schedule", "paged_kv_decode",
           "rotary_frequencies", "rotary_embedding", "rotary_paged_store", "rotary_paged_store8", "paged_kv8_read", "paged_kv8_decode", "paged_prefix_decode"]
