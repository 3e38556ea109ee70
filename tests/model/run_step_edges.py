"""A check of tests/step_edges.py on the CPU model of the library:

    python tests/model/run_step_edges.py <check>
"""

from __future__ import annotations

import os
import sys

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import run_step  # noqa: E402

if __name__ == "__main__":
    run_step.install()
    import step_edges
    step_edges.EDGES[sys.argv[1]]("cpu")
    print(f"{sys.argv[1]}: held", flush=True)
