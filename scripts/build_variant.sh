#!/bin/bash
# Build another copy of the HIP library with extra -D flags for within-run A/B measurements (load it with DIC_HIP_LIB=<path>):
#   scripts/build_variant.sh NAME "-DDIC_GEMM_WIDE_ORDER=0 -DDIC_CE_EXP_NT=0"   ->  abl/libdic_NAME.so   (abl/ travels to the GPU box, is not committed)
set -e
R=$(cd "$(dirname "$0")/.." && pwd)
NAME=$1; FLAGS=$2
mkdir -p $R/abl/obj_$NAME
cd $R
# one line per source: its compile command with the flags of the shipped build (_lib.py)
python - $R/abl/obj_$NAME $FLAGS > $R/abl/obj_$NAME/commands <<'END'
import importlib, os, shlex, sys
lib = importlib.import_module("diffusion-image-captioning_amd._lib")
for s in lib.SOURCES:
    print(shlex.join(lib.compile_command(s, os.path.join(sys.argv[1], s[:-4] + ".o"), sys.argv[2:])))
END
pids=""
n=0
while read -r cmd; do
  n=$((n + 1))
  eval "$cmd" 2> $R/abl/obj_$NAME/$n.log < /dev/null &
  pids="$pids $!"
done < $R/abl/obj_$NAME/commands
for p in $pids; do wait $p || { echo "build_variant.sh $NAME: a compile FAILED:"; grep -h -A3 "error" $R/abl/obj_$NAME/*.log | head -20; exit 1; }; done      # (a bare `wait` hides a failed compile: round 6 found a 0.5 MB "library" without its GEMMs)
${HIPCC:-/opt/rocm/bin/hipcc} --offload-arch=gfx950 -shared -fPIC -o $R/abl/libdic_$NAME.so $R/abl/obj_$NAME/*.o
rm -rf $R/abl/obj_$NAME
ls -la $R/abl/libdic_$NAME.so
