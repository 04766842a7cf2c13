"""B200-native decoder for lmz checkpoint archives.

`lmz_b200.gpu` mirrors the reference's `lmz.gpu` module (same function names,
arguments and error behaviour); `lmz_b200.archive` reads the reference's
archive layout and `lmz_b200.decode` drives whole-archive decode on the GPU;
`lmz_b200.embed`, `lmz_b200.adapters`, `lmz_b200.norms`, `lmz_b200.linear` and
`lmz_b200.experts` are operators on the tensors that come out.
Importing this package touches neither CUDA nor the compiler.
"""
__version__ = "0.1.0"
