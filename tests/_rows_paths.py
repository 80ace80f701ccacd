"""Sizes of the float products that go to kernels which smaller ones do not reach, each with the kernel's tile and the
slices of its sums (0: more than one)."""
FORWARD, SWIGLU, INPUT, WEIGHT = range(4)

# (dtype, in, out, tokens): ragged edges each way, more tiles than workgroups
LINEAR = [(("bf16", 136, 5128, 1990), 256, 1), (("f16", 264, 5128, 1990), 256, 1), (("f16", 136, 6152, 1333), 160, 1),
          (("bf16", 520, 6152, 1333), 160, 1), (("bf16", 136, 4104, 1333), 128, 1), (("f32", 72, 4104, 1333), 128, 1),
          (("f16", 2056, 264, 77), 64, 0)]
# ... of a weight's gradient, fp32 of 16 bits: two or three terms
WEIGHTS = [(("bf16", 4104, 2056, 333), 256, 1), (("f16", 4104, 2056, 333), 256, 1), (("f16", 4104, 2056, 100), 256, 1),
           (("bf16", 4104, 4104, 201), 128, 1), (("f16", 4104, 4104, 201), 128, 1), (("bf16", 264, 520, 2100), 64, 0),
           (("f16", 264, 520, 2100), 64, 0)]
# (dtype, hidden, intermediate, rows of each expert): the forward pass, and its weights' gradients
SWIGLU_FORWARD = [(("bf16", 2056, 2056, (300, 1, 0, 899)), 128, 1),
                  (("f16", 2056, 4104, (600, 500, 130, 1, 0, 1300, 900, 1069)), 256, 1),
                  (("bf16", 136, 2056, (300, 1, 0, 899)), 128, 1)]
SWIGLU_WEIGHTS = [(("bf16", 2056, 2056, (300, 1, 0, 899)), 256, 1), (("f16", 2056, 2056, (300, 1, 0, 899)), 256, 1),
                  (("f16", 136, 2056, (300, 1, 0, 899)), 128, 1), (("bf16", 136, 264, (70, 1, 0, 60)), 64, 1)]
