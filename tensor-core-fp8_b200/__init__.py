"""B200 (sm_100a) FP8 GEMM library -- Python host layer over the C ABI.

The directory name is not an identifier; import it through ``load_package()`` in
``__graft_entry__.py`` (it registers the package as ``tcfp8_b200``).

    from tcfp8_b200 import gemm        # GEMM / GEMM4: the reference's operator surface
    from tcfp8_b200 import shard       # N-sharded multi-GPU plan
    from tcfp8_b200 import experts     # products grouped by expert, their gradients, 4-bit weights (also names of gemm)
"""
from . import _cabi  # noqa: F401
from . import experts, gemm, shard  # noqa: F401

__all__ = ["gemm", "shard", "experts", "_cabi"]
