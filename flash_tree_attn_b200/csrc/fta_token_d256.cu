#define FTA_INST_D 256
#include "fta_token_stage1.inc"
