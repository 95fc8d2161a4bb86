"""The adapter pool's, the layer norm's and the orthogonalised step's argument
structs: ctypes mirrors, packed forms and header agree."""
import ctypes
import os
import shutil
import subprocess

import pytest

from foundry_attn import _abi

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "foundry_block.h")
STRUCTS = {"fa_layer_norm_args": _abi.LayerNormArgs, "fa_layer_norm_bwd_args": _abi.LayerNormBwdArgs,
           "fa_muon_args": _abi.MuonArgs, "fa_lora_pool_args": _abi.LoraPoolArgs,
           "fa_lora_pool_bwd_args": _abi.LoraPoolBwdArgs}


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not available")
def test_struct_layouts_match_header(tmp_path):
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void){"]
    for cname, py in STRUCTS.items():
        lines.append(f'printf("{cname} size %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname} {field} %zu\\n", offsetof({cname}, {field}));' for field, _ in py._fields_]
    lines += ['printf("limits rank %d\\n", FA_MUON_MAX_RANK);', 'printf("limits steps %d\\n", FA_MUON_MAX_STEPS);',
              "return 0;}"]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines))
    subprocess.run(["gcc", "-o", str(exe), str(src)], check=True)
    limits = {"rank": _abi.FA_MUON_MAX_RANK, "steps": _abi.FA_MUON_MAX_STEPS}
    for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines():
        cname, what, value = line.split()
        if cname == "limits":
            want = limits[what]
        elif what == "size":
            want = ctypes.sizeof(STRUCTS[cname])
        else:
            want = getattr(STRUCTS[cname], what).offset
        assert int(value) == want, (cname, what, value, want)
