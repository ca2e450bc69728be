"""linatt_b200 -- B200-native (sm_100a) KATA-SPD attention hot path of ayghri/linatt.

Drop-in modules mirroring the reference's operator API:
  linatt_b200.parallel_kata_attn   <-> kata/parallel_kata_attn.py
Generation (no counterpart in the reference):
  linatt_b200.generate   a KataLM on 4-bit weights and recurrent states, token by token
  linatt_b200.quant      linear layers with 4-bit weights and group scales
  linatt_b200.qkv_step   short convolution, head norms and rotation of one token
  linatt_b200.sampling   temperature, top-k, top-p and min-p from given random numbers
All compute runs in ``libkata_b200.so`` (C ABI: include/kata_b200.h); build it with
``python -m linatt_b200.build``.
"""

from ._lib import check_device_status  # noqa: F401

__all__ = ["check_device_status"]
