#!/bin/bash
# Experiment builds: libgnnrec with extra -D flags on ONE kernel source, linked from the
# in-tree objects of the others (run after build_native.py). Load with GNNREC_LIB=<out>.
#   bash tools/build_variant.sh <out.so> <source.hip> -DNAME=VALUE ...
set -euo pipefail
OUT=$1; SRC=$2; shift 2
B=gnn-recommendations_amd/build
mkdir -p "$(dirname "$OUT")"
T=$(mktemp -d)
HIPCC=${HIPCC:-/opt/rocm/bin/hipcc}
# the library's own flags: a variant differs from it by its -D flags alone
FLAGS=$(PYTHONPATH=gnn-recommendations_amd python3 -c \
  'import build_native; print(*build_native.CFLAGS)')
$HIPCC $FLAGS "$@" -c "gnn-recommendations_amd/csrc/$SRC" -o "$T/v.o"
OBJS=$(ls $B/*.o | grep -v "/$SRC.o$")
$HIPCC --offload-arch=gfx950 -shared -fPIC -o "$OUT" $OBJS "$T/v.o" -lpthread
rm -rf "$T"
echo "$OUT"
