"""yanchor_amd: MI355X-native kernels for YANchor's batched recurrent hot path.

Modules mirror the reference's call sites:

* ``yanchor_amd.gdn``                 gated delta rule (decode state update, chunked
                                      varlen prefill, drafted trees)
* ``yanchor_amd.independent_memory``  anchor memory read / commit
* ``yanchor_amd.inference_kernels``   counter sampling, presence penalty, slot
                                      bookkeeping, packing and compaction, block tables
* ``yanchor_amd.layers``              the steps between them: projections, norms,
                                      prefill, attention over drafted trees, quantised
                                      caches and the decode attention over them

All compute runs in hand-written HIP kernels from ``lib/libyanchor_amd.so``
(built by ``python -m yanchor_amd.build``); there is no CPU fallback.
"""
__version__ = "0.1.0"
