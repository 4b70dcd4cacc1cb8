"""Hand-written gfx950 HIP kernels: the synthetic load for the overhead benchmark (``load``) and the
decoder block's operators, forward and backward (``decoder``)."""
