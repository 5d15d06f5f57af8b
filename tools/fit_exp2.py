"""Coefficients of the 2^f polynomial in mpnn_amd/csrc/mpnn_beam.hip: interpolation at Chebyshev nodes of [-1/2, 1/2] in
extended precision (within a factor of two of the minimax error), printed with the error it has in fp64 Horner form."""
import sys

import numpy as np

degree = int(sys.argv[1]) if len(sys.argv) > 1 else 8
L = np.longdouble
k = np.arange(degree + 1, dtype=L)
nodes = np.cos((2 * k + 1) * L(np.pi) / (2 * (degree + 1))) / 2
V = np.stack([nodes**i for i in range(degree + 1)], 1)
# Newton's divided differences, then expansion to monomials: numpy's solvers have no extended precision
d = np.exp2(nodes)
for i in range(1, degree + 1):
    d[i:] = (d[i:] - d[i - 1:-1]) / (nodes[i:] - nodes[:-i])
c = np.zeros(degree + 1, dtype=L)
for i in range(degree, -1, -1):
    c = np.concatenate([[L(0)], c[:-1]]) - nodes[i] * c
    c[0] += d[i]
f = np.linspace(-0.5, 0.5, 200001).astype(np.float64)
y = np.full_like(f, float(c[-1]))
for a in c[-2::-1]:
    y = y * f + float(a)
ref = np.exp2(f.astype(L))
print("degree", degree, "max relative error %.2e" % float(np.max(np.abs((y - ref) / ref))))
for i, a in enumerate(c):
    print("c%d = %.17e" % (i, float(a)))
