"""Collective operations (module-level API), fused GEMM+collective ops, 8-bit formats and their products, and the LL128 layout oracle."""
