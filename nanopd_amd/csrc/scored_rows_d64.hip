// The rows kernel of the scored attention ops at padded head dim 64
// (scored_rows.h).
#include "scored_rows.h"

template void npd::scored::launch_rows<64>(const npd::scored::Args&, int32_t, hipStream_t);
