"""Write the golden outputs of the INT8 block's kernels (tests/block_inputs.py).

    python tests/golden/make_block_golden.py PACKAGE_DIR OUT_DIR

PACKAGE_DIR holds a built ``h3_speedkit`` whose kernels were compared bit for bit with the
reference's own (they need oracle/_ref, from the reference checkout); the files are what
later builds are held to where that checkout is absent.
"""
import sys
from pathlib import Path

import numpy as np
import torch

if __name__ == "__main__":
    package, out = Path(sys.argv[1]).resolve(), Path(sys.argv[2])
    sys.path[:0] = [str(package), str(Path(__file__).resolve().parents[1])]
    import block_inputs
    out.mkdir(parents=True, exist_ok=True)
    for name, arrays in block_inputs.outputs(torch.device("cuda", 0)).items():
        np.savez_compressed(out / f"{name}.npz", **arrays)
        print(name, {k: a.shape for k, a in arrays.items()})
