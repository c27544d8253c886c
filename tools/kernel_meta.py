"""Register / scratch / LDS figures of every kernel in the built library (from the gfx950 code objects embedded in libpocr_hip.so).
Usage: python tools/kernel_meta.py [substring filter]"""
import os, re, subprocess, sys, tempfile

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from codeobj_hash import code_objects  # noqa: E402

so = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "pero_ocr_amd", "libpocr_hip.so")
if len(sys.argv) > 2: so = sys.argv[2]
notes = ""
for elf in code_objects(so):                              # every translation unit's
    with tempfile.NamedTemporaryFile(suffix=".co") as f:
        f.write(elf); f.flush()
        notes += subprocess.run(["/opt/rocm/lib/llvm/bin/llvm-readelf", "--notes", f.name], capture_output=True, text=True, check=True).stdout
flt = sys.argv[1] if len(sys.argv) > 1 else ""
for blk in notes.split("- .agpr_count:")[1:]:
    g = lambda k: re.search(r"\." + k + r":\s*(\S+)", blk)
    nm = g("name").group(1)
    try:
        nm = subprocess.run(["/opt/rocm/lib/llvm/bin/llvm-cxxfilt", nm], capture_output=True, text=True).stdout.strip()
    except Exception:
        pass
    if flt in nm:
        print(f"vgpr {g('vgpr_count').group(1):>4} agpr {blk.split()[0]:>3} sgpr {g('sgpr_count').group(1):>4} scratch {g('private_segment_fixed_size').group(1):>4} lds {g('group_segment_fixed_size').group(1):>6}  {nm[:150]}")
