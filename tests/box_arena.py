"""A closed box as an arena mesh, for tests that need an env but no particular arena."""

from __future__ import annotations

from pathlib import Path

import numpy as np


def write_box(path: Path, cells: int = 4) -> Path:
    """8192 x 10240 x 2048 uu, each side `cells` x `cells` quads, normals inward; OBJ vertices are (y, x, z)."""
    lo, hi = np.array([-4096.0, -5120.0, 0.0]), np.array([4096.0, 5120.0, 2048.0])
    lines, faces, n = [], [], 0
    t = np.linspace(0.0, 1.0, cells + 1)
    for axis in range(3):
        u, v = (axis + 1) % 3, (axis + 2) % 3
        for side in (0, 1):
            for a in t:
                for b in t:
                    p = np.zeros(3)
                    p[axis] = (lo, hi)[side][axis]
                    p[u] = lo[u] + a * (hi[u] - lo[u])
                    p[v] = lo[v] + b * (hi[v] - lo[v])
                    lines.append(f"v {p[1]:.6f} {p[0]:.6f} {p[2]:.6f}")
            for i in range(cells):
                for j in range(cells):
                    q = [n + i * (cells + 1) + j, n + (i + 1) * (cells + 1) + j,
                         n + (i + 1) * (cells + 1) + j + 1, n + i * (cells + 1) + j + 1]
                    if side == 1:
                        q.reverse()
                    faces.append(f"f {q[0] + 1} {q[1] + 1} {q[2] + 1}")
                    faces.append(f"f {q[0] + 1} {q[2] + 1} {q[3] + 1}")
            n += (cells + 1) ** 2
    path.write_text("\n".join(lines + faces) + "\n")
    return path
