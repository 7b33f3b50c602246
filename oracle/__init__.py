"""CPU/PyTorch restatement of the reference encoder forward -- TEST INFRASTRUCTURE ONLY.

This package is the parity checker for the CUDA path in ``techjam_b200``.  Only
``tests/``, ``__graft_entry__.smoke()`` and ``bench.py``'s CPU-baseline leg may
import it, and only to *check* or to *time the reference arithmetic*; the
product path (``techjam_b200``) never imports, links or calls anything here.

Contents
--------
``reference_model``  the pre-LN encoder, the seeded input generator and the
                     OR-criterion checker, restated from the reference's
                     immutable ``torch_transformer_benchmark.py``.
``linear_memory``    the same model with attention evaluated in bounded-memory
                     FP32 chunks (for configurations whose dense score tensor
                     cannot be materialised), restated from
                     ``src/implementations/fp32_reference.py``.
``poly``             the chunked degree-2 polynomial linear attention and its
                     score-spread guard, restated from
                     ``src/implementations/poly_reference.py`` and
                     ``src/implementations/poly_guard.py``.
``act8``             8-bit activations and the training operators in 64 bits
                     (no counterpart in the reference).

Parity of this restatement is pinned by the golden fixtures in
``tests/golden/`` (generated by ``tests/golden/make_golden.py`` from the
reference's own modules) and checked by ``tests/test_oracle_golden.py``.
"""
